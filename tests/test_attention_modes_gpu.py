"""Gradients and refusals of SerializedAttention and of a block around it by mode: training, evaluation, autograd on and off."""
import pytest
import torch

import pointtransformerv3_b200 as P
from helpers import rel_l2
from test_attention_options_gpu import OPTIONS, module, reference, scene

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("name", [n for n in OPTIONS if n not in ("plain", "rpe")])
def test_gradients_in_evaluation(name, dtype):
    """A module with options beyond the reference's, frozen in evaluation mode: all gradients as in training mode, bit for bit, and
    without autograd none.  Bounds as for training: at most ten roundings of bf16, sums of fp32."""
    att = module(name, dtype, flash=True)
    pt, feat, dout = scene([300, 90], 51, 64, dtype)

    def run(training):
        att.train(training)
        x = feat.clone().requires_grad_()
        pt.feat = x
        out = att(pt).feat
        return (out.detach(),) + torch.autograd.grad(out, [x] + list(att.parameters()), dout)
    got = run(False)
    assert all(torch.equal(a, b) for a, b in zip(got, run(True)))
    want, _, dx = reference(att, pt, feat, dout)
    tol = 2e-5 if dtype == torch.float32 else 10 ** 0.5 * 2.0 ** -8
    assert rel_l2(got[0], want) < tol and rel_l2(got[1], dx) < tol
    att.eval()
    for p in att.parameters():
        p.requires_grad_(False)
    x = feat.clone().requires_grad_()                   # of the features alone
    pt.feat = x
    assert torch.equal(torch.autograd.grad(att(pt).feat, x, dout)[0], got[1])
    for p in att.parameters():
        p.requires_grad_(True)
    pt.feat = feat
    with torch.no_grad():
        out = att(pt).feat
    assert not out.requires_grad and rel_l2(out, want) < tol


def test_a_block_does_not_train_its_attention_alone():
    """Operators around the attention have no gradients, so a block in evaluation refuses an attention in training."""
    torch.manual_seed(0)
    block = P.Block(64, 4, 128, cpe_indice_key="s", upcast_attention=False, upcast_softmax=False,
                    attn_options=dict(qk_norm=True)).cuda().eval()
    pt, feat, _ = scene([200], 5, 64, torch.float32)
    pt.feat = feat
    pt.sparsify()
    with torch.no_grad():
        block(P.Point(dict(pt)))
    block.attn.train()
    with pytest.raises(AssertionError, match="inference only"):
        block(P.Point(dict(pt)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_a_bias_of_far_offsets_evaluates(dtype):
    """Patches of 10 000 have a bias for offsets up to 68, more than the inference kernel's table holds: what trains evaluates."""
    att = module("rpe", dtype, flash=False, K=10000)
    assert att.rpe.pos_bnd == 68
    pt, feat, dout = scene([300, 270], 61, 64, dtype)
    outs = []
    for training in (True, False):
        att.train(training)
        pt.feat = feat
        with torch.no_grad():
            outs.append(att(pt).feat)
    want = reference(att, pt, feat, dout)[0]
    for out in outs:
        assert rel_l2(out, want) < (2e-5 if dtype == torch.float32 else 10 ** 0.5 * 2.0 ** -8)
