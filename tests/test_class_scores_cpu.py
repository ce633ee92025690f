"""Scores of logits and losses against a teacher's lists, what needs no GPU: the 64-bit formulas against differentiation, and what the
entry points refuse before anything is launched."""
import math

import pytest
import torch

import class_scores_reference as R
from pointtransformerv3_b200 import _lib
from pointtransformerv3_b200 import functional as F

N, K = 9, 7


def normal(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


@pytest.mark.parametrize("temperature", [1.0, 0.5, 3.0])
def test_gradient_of_scores_is_the_derivative(temperature):
    x = (2 * normal(N, K, seed=1)).requires_grad_()
    labels = torch.arange(N) % (K + 1) - 1
    g, h, t = normal(N, seed=2), normal(N, seed=3), normal(N, 3, seed=4)
    logp = torch.log_softmax(x / temperature, 1)
    entropy = torch.distributions.Categorical(logits=logp).entropy()
    picked = torch.where(labels >= 0, logp.gather(1, labels.clamp_min(0)[:, None])[:, 0], 0.0)
    values, classes = logp.topk(3, 1)
    want = torch.autograd.grad((g * picked + h * entropy).sum() + (t * values).sum(), x)[0]
    out = R.scores(x.detach(), labels, 3, temperature, upstream=(g, h, t))
    for name, value in (("log_prob", picked), ("entropy", entropy), ("top_log_probs", values), ("dlogits", want)):
        assert torch.allclose(out[name][0], value.detach(), rtol=1e-12, atol=1e-13), name
    assert torch.equal(out["top_classes"][0], classes.int())
    # and differences
    step, e = 1e-6, torch.zeros(N, K, dtype=torch.float64)
    e[4, 2] = step

    def total(y):
        o = R.scores(y, labels, 3, temperature)
        return (g * o["log_prob"][0] + h * o["entropy"][0]).sum() + (t * o["top_log_probs"][0]).sum()
    slope = (total(x.detach() + e) - total(x.detach() - e)) / (2 * step)
    assert abs(slope - want[4, 2]) < 1e-7


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("temperature", [1.0, 2.5])
def test_gradient_of_a_list_is_the_derivative(rest, temperature):
    x = (2 * normal(N, K, seed=5)).requires_grad_()
    values, classes = torch.log_softmax(normal(N, K, seed=6), 1).topk(3, 1)
    classes[2] = -1
    classes[3, 1] = -1
    classes[4] = torch.tensor([1, 1, 5])            # a class twice
    there = classes >= 0
    at = classes.clamp_min(0)
    z = x / temperature
    if rest:
        t = torch.exp(values) * there
    else:
        t = torch.softmax(torch.where(there, values / temperature, -1e9), 1) * there
    logp = torch.log_softmax(z, 1)
    loss = (torch.xlogy(t, t) - t * logp.gather(1, at)).sum(1)
    if rest:
        member = torch.zeros(N, K).scatter_reduce(1, at, there.float(), "amax") > 0
        left = torch.where(there.any(1), 1 - t.sum(1), 0.0)
        p_r = torch.where(member, 0.0, torch.exp(logp)).sum(1)
        loss = loss + torch.xlogy(left, left) - left * torch.log(p_r)
    g = normal(N, seed=7)
    want = torch.autograd.grad((g * loss).sum(), x)[0]
    out = R.distill(x.detach(), values, classes, temperature, rest, upstream=g)
    assert torch.allclose(out["loss"][0], loss.detach(), rtol=1e-12, atol=1e-13)
    assert torch.allclose(out["dlogits"][0], want, rtol=1e-12, atol=1e-13)


def test_reference_of_rows_that_masks_empty():
    x = torch.full((4, 5), -math.inf)
    x[1, 3] = 2.0
    x[2, :] = torch.finfo(torch.float32).min
    x[3, 1] = math.nan
    out = R.scores(x, torch.tensor([0, 3, 4, 2]), 2, upstream=(torch.ones(4), torch.ones(4), None))
    assert out["log_prob"][0][:3].tolist() == [-math.inf, 0.0, -math.log(5)] and out["log_prob"][0][3].isnan()
    assert out["entropy"][0][:2].tolist() == [0, 0] and abs(out["entropy"][0][2] - math.log(5)) < 1e-12
    assert out["top_classes"][0].tolist() == [[0, 1], [3, 0], [0, 1], [1, 0]]
    assert (out["dlogits"][0][0] == 0).all()
    lists = torch.tensor([[1, 2]] * 4)
    out = R.distill(x, torch.zeros(4, 2), lists, upstream=torch.ones(4))
    assert out["loss"][0][:2].tolist() == [math.inf, math.inf] and (out["dlogits"][0][0] == 0).all()


ROWS, WORD = 1 << 20, 1 << 21      # made-up addresses: nothing is launched


def scores_fwd(logits=ROWS, ld=20, labels=ROWS, label_bytes=8, ignore=-1, log_prob=ROWS, entropy=ROWS, values=ROWS, classes=ROWS,
               stats=None, n=4, K=20, top=3, temperature=1.0, dtype=0, status=WORD):
    return _lib.load().ptv3_class_scores_fwd(logits, ld, labels, label_bytes, ignore, log_prob, entropy, values, classes, stats, n, K, top,
                                             temperature, dtype, status, None)


def scores_bwd(logits=ROWS, ld=20, labels=ROWS, label_bytes=8, classes=ROWS, stats=ROWS, g=ROWS, h=ROWS, t=ROWS,
               dlogits=ROWS, n=4, K=20, top=3, temperature=1.0, dtype=0):
    return _lib.load().ptv3_class_scores_bwd(logits, ld, labels, label_bytes, -1, classes, stats, g, 1, h, 1, t, dlogits, n, K, top,
                                             temperature, dtype, None)


def distill_fwd(logits=ROWS, ld=20, teacher=ROWS, teacher_dtype=0, classes=ROWS, size=4, k=3, loss=ROWS, stats=None, n=4, K=20,
                temperature=1.0, rest=0, dtype=0, status=WORD):
    return _lib.load().ptv3_distill_topk_fwd(logits, ld, teacher, teacher_dtype, classes, size, k, loss, stats, n, K, temperature, rest, dtype,
                                             status, None)


def distill_bwd(logits=ROWS, ld=20, teacher=ROWS, classes=ROWS, size=4, k=3, stats=ROWS, g=ROWS, dlogits=ROWS, n=4, K=20,
                temperature=1.0, rest=0, dtype=0):
    return _lib.load().ptv3_distill_topk_bwd(logits, ld, teacher, 0, classes, size, k, stats, g, 1, dlogits, n, K, temperature, rest, dtype, None)


def head(feat=ROWS, weight=ROWS, bias=ROWS, labels=ROWS, label_bytes=8, log_prob=ROWS, entropy=ROWS, values=ROWS, classes=ROWS, n=4, C=64, K=20,
         top=3, temperature=1.0, dtype=1, status=WORD):
    return _lib.load().ptv3_seg_head_scores_fwd(feat, weight, bias, labels, label_bytes, -1, log_prob, entropy, values, classes, n, C, K, top,
                                                temperature, dtype, status, None)


SHARED = [dict(n=-1), dict(n=2 ** 31), dict(dtype=2), dict(K=0), dict(K=2 ** 18 + 1, ld=2 ** 19), dict(ld=19), dict(temperature=0.0),
          dict(temperature=-1.0), dict(temperature=math.nan), dict(temperature=math.inf), dict(logits=None), dict(logits=ROWS + 2)]
REFUSED = {
    scores_fwd: SHARED + [dict(top=-1), dict(top=65), dict(label_bytes=2), dict(labels=None), dict(values=None), dict(classes=None),
                          dict(status=None), dict(stats=ROWS + 4), dict(dtype=1, logits=ROWS + 1), dict(labels=ROWS + 4), dict(values=ROWS + 2),
                          dict(entropy=ROWS + 1)],
    scores_bwd: SHARED + [dict(top=65), dict(stats=None), dict(dlogits=None), dict(labels=None), dict(classes=None), dict(stats=ROWS + 8),
                          dict(dlogits=ROWS + 2), dict(label_bytes=1), dict(g=ROWS + 2), dict(labels=ROWS + 2, label_bytes=4)],
    distill_fwd: SHARED + [dict(k=0), dict(k=65), dict(teacher_dtype=2), dict(size=2), dict(teacher=None), dict(classes=None), dict(loss=None),
                           dict(status=None), dict(teacher=ROWS + 2), dict(classes=ROWS + 4, size=8), dict(stats=ROWS + 8), dict(loss=ROWS + 2)],
    head: [dict(n=-1), dict(n=2 ** 31 - 1), dict(dtype=0), dict(K=0), dict(K=2 ** 18 + 1), dict(C=0), dict(C=60), dict(C=520), dict(top=-1),
           dict(top=33), dict(temperature=0.0), dict(temperature=math.nan), dict(label_bytes=2), dict(labels=None), dict(feat=None),
           dict(weight=None), dict(entropy=None), dict(values=None), dict(classes=None), dict(status=None), dict(feat=ROWS + 8),
           dict(weight=ROWS + 2), dict(bias=ROWS + 1), dict(labels=ROWS + 4), dict(entropy=ROWS + 2)],
    distill_bwd: SHARED + [dict(k=0), dict(stats=None), dict(g=None), dict(dlogits=None), dict(dlogits=ROWS + 2)],
}


@pytest.mark.parametrize("call,wrong", [(f, w) for f, ws in REFUSED.items() for w in ws], ids=lambda v: getattr(v, "__name__", str(v)))
def test_refused_before_a_launch(call, wrong):
    assert call(**wrong) < 0
    assert call.__name__.split("_")[0] in _lib.load().ptv3_last_error().decode()


def test_no_rows_are_no_launch():
    before = _lib.load().ptv3_launch_count()
    for call in REFUSED:
        assert call(n=0) == 0
    assert _lib.load().ptv3_launch_count() == before


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 5)
    with pytest.raises(_lib.Ptv3Error, match="CUDA"):
        F.class_log_probs(x)
    with pytest.raises(_lib.Ptv3Error, match="CUDA"):
        F.distill_topk(x, torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int32))
