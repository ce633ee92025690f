"""The operators behind the logits with rows enough for a tile on every multiprocessor, where longer rows lie in tiles too: the inputs of the tests of few
rows, again and again, against the formulas in 64 bits."""
import pytest
import torch

import class_scores_reference as R
import test_class_scores_gpu as S
import test_distill_gpu as D
from pointtransformerv3_b200 import ops
from pointtransformerv3_b200 import functional as F

pytestmark = pytest.mark.gpu

MANY = 148 * 128 + 1


def again(t):
    return None if t is None else t.repeat(MANY // t.shape[0] + 1, *[1] * (t.dim() - 1))


def near(got, want, name):
    """Every copy (a row that starts elsewhere is summed in another order)."""
    value, tolerance = want
    R.assert_near(got, again(value), again(tolerance) if torch.is_tensor(tolerance) and tolerance.dim() else tolerance, name)


def check_scores(x, labels=None, top=0, temperature=1.0, ignore_index=-1, upstream=None, status=None):
    want = R.scores(x, labels, top, temperature, ignore_index, upstream)
    leaf = again(x).requires_grad_()
    out = F.class_log_probs(leaf, again(labels), top, temperature, ignore_index, ops.new_status("cuda"))
    for name in ("log_prob", "entropy", "top_log_probs"):
        if name in want:
            near(getattr(out, name).detach(), want[name], name)
    if top:
        assert torch.equal(out.top_classes, again(want["top_classes"][0]))
    pairs = [(o, again(u)) for o, u in zip(out[:3], upstream) if u is not None]
    dx = torch.autograd.grad([p[0] for p in pairs], leaf, [p[1] for p in pairs])[0]
    near(dx, want["dlogits"], "dlogits")


def check_distill(x, values, classes, temperature=1.0, rest=False, status=None, upstream=True):
    n = x.shape[0]
    g = D.normal(n, seed=77)
    want = R.distill(x, values, classes, temperature, rest, g)
    leaf = again(x).requires_grad_()
    loss = F.distill_topk(leaf, again(values), again(classes), temperature, rest, ops.new_status("cuda"))
    near(loss.detach(), want["loss"], "loss")
    near(torch.autograd.grad(loss, leaf, again(g))[0], want["dlogits"], "dlogits")
    return loss.detach()[:n]


@pytest.mark.parametrize("dtype", S.DTYPES, ids=["fp32", "bf16"])
@pytest.mark.parametrize("K", [33, 40, 65, 72, 80, 81, 128, 129, 166, 176, 177, 256, 257, 333, 352, 353, 500, 511, 512, 513])
def test_scores(K, dtype, monkeypatch):
    monkeypatch.setattr(S, "check", check_scores)
    x = S.normal(131, K, seed=K, scale=2.0, dtype=dtype)
    for top in (0, (1, 2, 3, 8)[K % 4], (16, 17, 32, 33)[K % 4]):
        S.check(x, S.labels_of(131, K, K), top, (1.0, 0.5, 3.0)[K % 3], upstream=S.upstream_of(131, top))


@pytest.mark.parametrize("dtype", S.DTYPES, ids=["fp32", "bf16"])
@pytest.mark.parametrize("K", [150, 352, 500])
def test_scores_beyond_the_ordinary(K, dtype, monkeypatch):
    monkeypatch.setattr(S, "check", check_scores)
    S.test_rows_beyond_the_ordinary(K, dtype)
    S.test_equal_logits_go_to_the_lowest_class(K, dtype)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype", S.DTYPES, ids=["fp32", "bf16"])
@pytest.mark.parametrize("K", [33, 40, 65, 72, 128, 166, 176, 177, 256, 300, 333, 352, 353])
def test_losses(K, dtype, rest):
    for k in ((1, 4, 5, 8)[K % 4], (9, 16, 17, 31)[K % 4], 32, 33):
        values, classes = D.teacher_of(131, K, k, rest, 2.0, K, torch.float32 if rest else dtype)
        check_distill(D.normal(131, K, seed=K + 1, scale=2.0, dtype=dtype), values, classes.long() if K % 2 else classes, 2.0, rest)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("K", [90, 176, 350])
def test_losses_beyond_the_ordinary(K, rest, monkeypatch):
    monkeypatch.setattr(D, "check", check_distill)
    D.test_lists_beyond_the_ordinary(K, rest)
    for dtype in S.DTYPES:
        D.test_students_beyond_the_ordinary(K, rest, dtype)


@pytest.mark.parametrize("K", [64, 150])
def test_long_lists_with_a_class_twice(K):
    """Of 32 entries in a tile: the first and the last alike, all alike, every other one absent."""
    for rest in (False, True):
        values, classes = D.teacher_of(12, K, 32, rest, 1.0, 3)
        classes[0, 31] = classes[0, 0]
        classes[1] = classes[1, 5]
        values[1] -= 4.0
        classes[2, 1::2] = -1
        classes[3] = -1
        classes[4, 20:] = classes[4, 10]
        for dtype in S.DTYPES:
            check_distill(D.normal(12, K, seed=5, scale=2.0, dtype=dtype), values, classes, 1.0, rest)
