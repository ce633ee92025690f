"""Log probabilities, entropy and alternatives of logits, and their gradients, against the formulas in 64 bits."""
import math

import pytest
import torch

import class_scores_reference as R
from pointtransformerv3_b200 import _lib, ops
from pointtransformerv3_b200 import functional as F

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]
INF = math.inf


def normal(*shape, seed, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def labels_of(n, K, seed=0, dtype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-1, K, (n,), generator=g).to(dtype).cuda()


def check(x, labels=None, top=0, temperature=1.0, ignore_index=-1, upstream=None, status=None):
    """Forward without and with gradients, and the gradient, against the reference."""
    if status is None:
        status = ops.new_status("cuda")
    plain = F.class_log_probs(x, labels, top, temperature, ignore_index, status)
    want = R.scores(x, labels, top, temperature, ignore_index, upstream)
    assert (plain.log_prob is None) == (labels is None) and (plain.top_classes is None) == (top == 0)
    for name in ("log_prob", "entropy", "top_log_probs"):
        if name in want:
            R.assert_near(getattr(plain, name), *want[name], name)
    if top:
        assert plain.top_classes.dtype == torch.int32 and torch.equal(plain.top_classes, want["top_classes"][0]), "top_classes"
    if upstream is not None:
        leaf = x.detach().requires_grad_()
        out = F.class_log_probs(leaf, labels, top, temperature, ignore_index, status)
        for a, b in zip(out, plain):
            assert (a is None and b is None) or torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))
        pairs = [(o, u) for o, u in zip(out[:3], upstream) if u is not None]
        dx = torch.autograd.grad([p[0] for p in pairs], leaf, [p[1] for p in pairs])[0]
        assert dx.dtype == x.dtype and dx.shape == x.shape
        R.assert_near(dx, *want["dlogits"], "dlogits")
    return plain


def upstream_of(n, top, seed=3):
    return normal(n, seed=seed), normal(n, seed=seed + 1, scale=0.5), normal(n, top, seed=seed + 2) if top else None


CLASSES = [1, 2, 3, 13, 20, 31, 32, 33, 63, 64, 65, 72, 100, 200, 255, 256, 257, 333, 512, 513, 1000, 1024, 1025, 1201, 2048, 2049,
           4097, 8192, 8200, 20001]


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16"])
@pytest.mark.parametrize("K", CLASSES)
def test_scores_and_gradients(K, dtype):
    n = 131 if K <= 1024 else 9
    top = (0, 1, 4, 7, 16, 32, 64)[K % 7]
    x = normal(n, K, seed=K, scale=2.0, dtype=dtype)
    check(x, labels_of(n, K, K, torch.int32 if K % 2 else torch.int64), top, (1.0, 0.5, 3.0)[K % 3], upstream=upstream_of(n, top))


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16"])
@pytest.mark.parametrize("n", [1, 2, 127, 128, 129, 1000])
def test_numbers_of_rows(n, dtype):
    for K in (20, 96, 1500):
        check(normal(n, K, seed=n, dtype=dtype), labels_of(n, K), 3, upstream=upstream_of(n, 3))


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16"])
@pytest.mark.parametrize("top", [1, 2, 3, 4, 5, 8, 9, 16, 17, 31, 32, 33, 63, 64])
def test_numbers_of_alternatives(top, dtype):
    """Also more than there are classes: minus infinity and no class."""
    for K in (1, 5, 40, 64, 66, 300, 1100, 3001):
        x = normal(21, K, seed=top, dtype=dtype)
        check(x, None, top, upstream=(None, None, normal(21, top, seed=5)))


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16"])
@pytest.mark.parametrize("K", [6, 50, 64, 150, 600, 1030, 2500, 9000])
def test_equal_logits_go_to_the_lowest_class(K, dtype):
    n = 40
    g = torch.Generator().manual_seed(K)
    x = torch.randint(-2, 3, (n, K), generator=g).float()
    x[0] = 0.25
    x[1] = torch.finfo(dtype).min
    x[2] = torch.where(torch.arange(K) % 2 == 0, -0.0, 0.0)
    x[3] = -1.0
    x[3, K - 2:] = 1.0
    x[4] = torch.arange(K) // 3 % 5
    x[5] = -INF
    x[6] = -INF
    x[6, K // 2] = -3.0
    for top in (1, 5, 33):
        check(x.to(dtype).cuda(), labels_of(n, K), top, upstream=upstream_of(n, top))


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16"])
@pytest.mark.parametrize("K", [7, 64, 130, 1024, 1100, 10000])
def test_rows_beyond_the_ordinary(K, dtype):
    """Masked classes, rows of masks alone, the type's lowest and largest values, far offsets, infinities and NaN."""
    n = 64
    x = normal(n, K, seed=K)
    low = torch.finfo(dtype).min
    x[0] = -INF
    x[1] = low
    x[2, 1:] = -INF
    x[3, :K - 1] = low
    x[4] += 30000.0
    x[5] -= 30000.0
    x[6, 2] = math.nan
    x[7, 3] = INF
    x[8, 3], x[8, 4] = INF, -INF
    x[9] = math.nan
    x[10, 0], x[10, 1] = torch.finfo(dtype).max, low
    x[11] = torch.finfo(dtype).max
    x[12] = -INF
    x[12, K - 1] = math.nan
    x[13] = 1e-42                       # below the smallest normal number
    x[13, 2] = 2e-42
    x[14, ::2] = -INF
    x[15] *= 40
    x[16, 5] += 12
    x[17, 5] += 90
    x = x.to(dtype)
    labels = labels_of(n, K)
    labels[2] = 0
    labels[14] = 0                      # masked
    labels[15] = 1
    for temperature in (1.0, 0.25):
        check(x, labels, 4, temperature, upstream=upstream_of(n, 4))


@pytest.mark.parametrize("which", range(1, 8))
@pytest.mark.parametrize("K", [20, 70, 1050])
def test_each_set_of_gradients(which, K):
    up = upstream_of(33, 5)
    check(normal(33, K, seed=1), labels_of(33, K), 5, upstream=tuple(u if which >> i & 1 else None for i, u in enumerate(up)))


@pytest.mark.parametrize("K", [20, 70, 1050])
def test_gradients_that_are_one_value_for_all_rows(K):
    x = normal(50, K, seed=2).requires_grad_()
    labels = labels_of(50, K)
    status = ops.new_status("cuda")
    out = F.class_log_probs(x, labels, 2, status=status)
    got = torch.autograd.grad(out.log_prob.sum() * 2 + out.entropy.mean() + out.top_log_probs.sum(), x)[0]
    ones = torch.ones(50, device="cuda")
    want = R.scores(x.detach(), labels, 2, upstream=(2 * ones, ones / 50, torch.ones(50, 2, device="cuda")))
    R.assert_near(got, *want["dlogits"], "dlogits")
    # steps between the gradients' values
    g = normal(50, 3, seed=3)
    out = F.class_log_probs(x, labels, 2, status=status)
    got = torch.autograd.grad((out.log_prob, out.entropy), x, (g[:, 1], g[:, 2]))[0]
    R.assert_near(got, *R.scores(x.detach(), labels, upstream=(g[:, 1], g[:, 2], None))["dlogits"], "dlogits")


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16"])
def test_rows_of_wider_ones_and_other_strides(dtype):
    """A slice is read where it is, whatever its alignment; other orders are copied."""
    for n, K, first, width in ((130, 20, 0, 24), (130, 20, 3, 25), (65, 200, 8, 216), (65, 200, 1, 208), (9, 1200, 5, 1211), (1, 96, 7, 200)):
        wide = normal(n, width, seed=K, dtype=dtype)
        check(wide[:, first:first + K], labels_of(n, K), 4, upstream=upstream_of(n, 4))
    check(normal(20, 33, seed=1, dtype=dtype).t(), labels_of(33, 20), 4, upstream=upstream_of(33, 4))
    check(normal(1, 33, seed=1, dtype=dtype).expand(40, 33), labels_of(40, 33), 4, upstream=upstream_of(40, 4))
    check(normal(40, 66, seed=1, dtype=dtype)[:, ::2], labels_of(80, 33)[::2], 4, upstream=upstream_of(40, 4))
    check(normal(40, 9, seed=1, dtype=dtype)[:, 4:5], labels_of(40, 1), 2, upstream=upstream_of(40, 2))


@pytest.mark.parametrize("K", [20, 100, 1100])
def test_labels(K):
    x = normal(60, K, seed=4)
    for ignore in (-1, -100, 0, 255, 3, 2 ** 40):
        labels = torch.randint(0, K, (60,), generator=torch.Generator().manual_seed(1)).cuda()
        labels[::7] = ignore
        check(x, labels, 0, ignore_index=ignore, upstream=upstream_of(60, 0))
    # out of range: NaN, a bit of the status word, no part of the gradient
    for wrong in (-1, -2, K, K + 5, 2 ** 40 + 1, -2 ** 63, 2 ** 63 - 1):
        labels = torch.zeros(60, dtype=torch.int64, device="cuda")
        labels[17] = wrong
        status = ops.new_status("cuda")
        out = check(x, labels, 0, ignore_index=-100, upstream=upstream_of(60, 0), status=status)
        assert int(status) == 1 and int(out.log_prob.isnan().sum()) == 1
        with pytest.raises(_lib.Ptv3Error, match="out of range"):
            F.class_log_probs(x, labels, ignore_index=-100)
    assert F.class_log_probs(x, torch.zeros(60, dtype=torch.int32, device="cuda")).log_prob.shape == (60,)


def test_no_points():
    for dtype in DTYPES:
        x = torch.empty(0, 20, device="cuda", dtype=dtype, requires_grad=True)
        out = F.class_log_probs(x, torch.empty(0, dtype=torch.int64, device="cuda"), 3)
        assert out.log_prob.shape == out.entropy.shape == (0,) and out.top_classes.shape == (0, 3)
        assert torch.autograd.grad(out.log_prob.sum(), x)[0].shape == (0, 20)


def test_rows_behind_four_gigabytes():
    """Offsets that pass 32 bits: the last rows of a long matrix, and of its gradient."""
    n, K = 33000, 2 ** 17
    x = torch.zeros(n, K, device="cuda", dtype=torch.bfloat16)
    x[-3:] = normal(3, K, seed=1, dtype=torch.bfloat16)
    labels = torch.full((n,), 5, device="cuda")
    want = R.scores(x[-3:], labels[-3:], 5, upstream=(torch.ones(3, device="cuda"), None, None))
    x.requires_grad_()
    out = F.class_log_probs(x, labels, 5)
    for name in ("log_prob", "entropy", "top_log_probs"):
        R.assert_near(getattr(out, name)[-3:], *want[name], name)
    assert torch.equal(out.top_classes[-3:], want["top_classes"][0])
    dx = torch.autograd.grad(out.log_prob, x, torch.ones(n, device="cuda"))[0]
    R.assert_near(dx[-3:], *want["dlogits"], "dlogits")


def test_the_most_classes():
    K = F.CLASSES_MAX
    x = normal(2, K, seed=9)
    check(x, labels_of(2, K), 64, upstream=upstream_of(2, 64))
    with pytest.raises(ValueError, match="classes"):
        F.class_log_probs(torch.zeros(1, K + 1, device="cuda"))


@pytest.mark.parametrize("K", [20, 200, 1500])
def test_other_streams_and_graphs(K):
    x, labels = normal(300, K, seed=6, dtype=torch.bfloat16), labels_of(300, K)
    status = ops.new_status("cuda")
    up = normal(300, seed=7)

    def step(x):
        leaf = x.detach().requires_grad_()
        out = F.class_log_probs(leaf, labels, 3, status=status)
        return [t.detach() for t in out] + [torch.autograd.grad(out.log_prob, leaf, up)[0]]
    want = step(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    held = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(held)
    held.copy_(normal(300, K, seed=8, dtype=torch.bfloat16))
    want = step(held)
    graph.replay()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(ValueError, match="status"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            F.class_log_probs(held, labels)
    assert int(status) == 0


def test_refusals():
    x = torch.zeros(4, 6, device="cuda")
    lab = torch.zeros(4, dtype=torch.int64, device="cuda")
    for args, kw, word in (((x[0],), {}, "logits"), ((x[:, :0],), {}, "logits"), ((x, lab[:3]), {}, "labels"),
                           ((x, lab.float()), {}, "labels"), ((x, lab.to(torch.int16)), {}, "labels"), ((x,), dict(top=-1), "alternatives"),
                           ((x,), dict(top=65), "alternatives"), ((x,), dict(temperature=0.0), "temperature"),
                           ((x,), dict(temperature=math.nan), "temperature"), ((x,), dict(temperature=-2.0), "temperature"),
                           ((x, lab), dict(status=torch.zeros(1, device="cuda")), "status"),
                           ((x, lab), dict(ignore_index=2 ** 63), "ignore_index")):
        with pytest.raises(ValueError, match=word):
            F.class_log_probs(*args, **kw)
    for dtype in (torch.float16, torch.float64):
        with pytest.raises(_lib.Ptv3Error, match="not supported"):
            F.class_log_probs(x.to(dtype))
    with pytest.raises(_lib.Ptv3Error, match="CUDA"):
        F.class_log_probs(x, lab.cpu())
    leaf = x.clone().requires_grad_()
    out = F.class_log_probs(leaf, lab)
    grad = torch.autograd.grad(out.log_prob.sum(), leaf, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        grad.sum().backward()
    with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError):
        F.class_log_probs(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)))


def test_labels_made_in_inference_mode_and_changed_ones():
    with torch.inference_mode():
        lab = torch.zeros(4, dtype=torch.int64, device="cuda")
    x = normal(4, 6, seed=1).requires_grad_()
    torch.autograd.grad(F.class_log_probs(x, lab).log_prob.sum(), x)
    lab = torch.zeros(4, dtype=torch.int64, device="cuda")
    out = F.class_log_probs(x, lab)
    lab += 1
    with pytest.raises(RuntimeError, match="modified"):
        torch.autograd.grad(out.log_prob.sum(), x)


@pytest.mark.parametrize("K", [20, 333, 1201])
def test_the_same_bits_on_every_run(K):
    x, labels = normal(500, K, seed=6, dtype=torch.bfloat16), labels_of(500, K)

    def step():
        leaf = x.detach().requires_grad_()
        out = F.class_log_probs(leaf, labels, 8)
        return list(out) + list(torch.autograd.grad(out[:3], leaf, upstream_of(500, 8)))
    first = step()
    assert all(torch.equal(a, b) for _ in range(3) for a, b in zip(first, step()))
