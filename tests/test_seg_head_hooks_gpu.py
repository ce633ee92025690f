"""A segmentation head whose layer has hooks: scores are those of the layer as a call of it is, not of a weight that an earlier call left."""
import pytest
import torch
from torch import nn

import class_scores_reference as R
from pointtransformerv3_b200 import SegHead

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore:.*weight_norm.*is deprecated")]


@torch.no_grad()
def normed(by):
    """A head in bf16 whose weight a hook makes, after a call and a change of what it is made from; features; the weight before, and as it is now in
    64 bits; how many half steps of bf16 that one is off by at most."""
    torch.manual_seed(0)
    head = SegHead(64, 20).cuda().bfloat16()
    feat = torch.randn(300, 64, device="cuda").bfloat16()
    layer = head.linear
    if by == "weight_norm":
        nn.utils.weight_norm(layer)
    else:
        nn.utils.spectral_norm(layer)
        u, _, v = torch.linalg.svd(layer.weight_orig.float())
        layer.weight_u.copy_(u[:, 0])
        layer.weight_v.copy_(v[0])
    head.eval()
    layer(feat)
    before = layer.weight.double()
    if by == "weight_norm":
        layer.weight_g.mul_(-2)
        v = layer.weight_v.double()
        return head, feat, before, layer.weight_g.double() * v / v.norm(dim=1, keepdim=True), 4        # norm, quotient, factor, product
    layer.weight_orig.copy_(layer.weight_orig.flip(0))
    layer.weight_u.copy_(layer.weight_u.flip(0))
    w, u = layer.weight_orig.double(), layer.weight_u.double()
    wv = w @ layer.weight_v.double()
    sigma = u @ wv
    # W v, its product with u, the quotient; the first two as far as they cancel
    return head, feat, before, w / sigma, 1 + 2 * float((u.abs() @ wv.abs()) / sigma.abs())


def near(got, logits, eps, **kw):
    """Log probabilities of logits that are off by at most eps each: by twice that."""
    want = R.scores(logits, **kw)
    for name in ("log_prob", "top_log_probs"):
        if name in want:
            R.assert_near(getattr(got, name), want[name][0], want[name][1] + 2 * eps, name)


@pytest.mark.parametrize("by", ["weight_norm", "spectral_norm"])
@torch.no_grad()
def test_weights_that_a_hook_makes(by):
    head, feat, before, weight, halves = normed(by)
    labels = torch.arange(300, device="cuda") % 20
    got = head.log_probs(feat, labels, top=3)
    bias = head.linear.bias.double()
    logits = feat.double() @ weight.t() + bias
    half = torch.finfo(torch.bfloat16).eps / 2
    eps = float(half * (1.1 * halves * (feat.double().abs() @ weight.abs().t()).max() + 1.1 * logits.abs().max()))
    near(got, logits, eps, labels=labels, top=3)
    stale = R.scores(feat.double() @ before.t() + bias, labels)["log_prob"][0]
    assert (stale - R.scores(logits, labels)["log_prob"][0]).abs().max() > 4 * eps


@pytest.mark.parametrize("kind", ["forward", "pre", "global"])
def test_hooks_of_the_layer_run(kind):
    """What a hook does to the layer's input or output is in the scores, and it is called."""
    torch.manual_seed(0)
    head = SegHead(64, 20).cuda().bfloat16()
    feat = torch.randn(300, 64, device="cuda").bfloat16()
    calls = []

    def after(module, args, out):
        if module is head.linear:
            calls.append(1)
            return out * 0

    def before(module, args):
        calls.append(1)
        return (args[0] * 0,)
    if kind == "forward":
        handle = head.linear.register_forward_hook(after)
    elif kind == "pre":
        handle = head.linear.register_forward_pre_hook(before)
    else:
        handle = nn.modules.module.register_module_forward_hook(after)
    try:
        with torch.no_grad():
            got = head.log_probs(feat, top=2)
    finally:
        handle.remove()
    assert calls == [1]
    logits = (head.linear.bias.detach() if kind == "pre" else torch.zeros(20, device="cuda").bfloat16()).expand(300, 20)
    near(got, logits.double(), 0.0, top=2)
    with torch.no_grad():
        assert not torch.equal(head.log_probs(feat, top=2).top_log_probs, got.top_log_probs)
