"""A student's loss against a teacher's lists, and its gradient, against the formulas in 64 bits."""
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


def teacher_of(n, K, k, rest, temperature, seed=0, dtype=torch.float32, peak=2.0):
    """Lists of k entries, those beyond the classes absent."""
    t = normal(n, K, seed=seed, scale=peak) / temperature
    out = F.class_log_probs(t, top=k) if rest else t.topk(min(k, K), 1)
    values, classes = (out.top_log_probs, out.top_classes) if rest else out
    if values.shape[1] < k:
        values = torch.nn.functional.pad(values, (0, k - K), value=-INF)
        classes = torch.nn.functional.pad(classes, (0, k - K), value=-1)
    return values.to(dtype), classes


def check(x, values, classes, temperature=1.0, rest=False, status=None, upstream=True):
    if status is None:
        status = ops.new_status("cuda")
    g = normal(x.shape[0], seed=77) if upstream is True else upstream
    want = R.distill(x, values, classes, temperature, rest, g)
    plain = F.distill_topk(x, values, classes, temperature, rest, status)
    R.assert_near(plain, *want["loss"], "loss")
    leaf = x.detach().requires_grad_()
    loss = F.distill_topk(leaf, values, classes, temperature, rest, status)
    assert torch.equal(loss.nan_to_num(7.0), plain.nan_to_num(7.0))
    dx = torch.autograd.grad(loss, leaf, g)[0]
    assert dx.dtype == x.dtype and dx.shape == x.shape
    R.assert_near(dx, *want["dlogits"], "dlogits")
    return plain


CLASSES = [1, 2, 3, 13, 20, 31, 32, 33, 63, 64, 65, 72, 100, 200, 256, 333, 512, 513, 1000, 1024, 1025, 1201, 2048, 2049, 8192, 8193, 20001]


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16"])
@pytest.mark.parametrize("K", CLASSES)
def test_losses_and_gradients(K, dtype, rest):
    n = 131 if K <= 1024 else 9
    k = (1, 4, 8, 16, 33, 64)[K % 6]
    temperature = (1.0, 0.5, 3.0)[K % 3]
    values, classes = teacher_of(n, K, k, rest, temperature, K)
    check(normal(n, K, seed=K + 1, scale=2.0, dtype=dtype), values, classes.long() if K % 2 else classes, temperature, rest)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("n", [1, 2, 127, 128, 129, 1000])
def test_numbers_of_rows(n, rest):
    for K in (20, 96, 1500):
        check(normal(n, K, seed=n), *teacher_of(n, K, 5, rest, 1.0, n), rest=rest)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("k", [1, 2, 7, 8, 31, 32, 33, 63, 64])
def test_lengths_of_lists(k, rest):
    """Also lists that hold every class, and lists longer than that."""
    for K in (1, 5, 32, 64, 66, 300, 1100):
        check(normal(21, K, seed=k), *teacher_of(21, K, k, rest, 1.0, k, torch.bfloat16 if k % 2 and not rest else torch.float32), rest=rest)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("K", [12, 64, 90, 1500])
def test_lists_beyond_the_ordinary(K, rest):
    """Absent entries, rows of them, a class twice, entries of no probability, orders other than by size, certain teachers."""
    n, k = 40, 6
    values, classes = teacher_of(n, K, k, rest, 1.0, 3)
    classes[0] = -1
    classes[1, 1:] = -1
    classes[2, ::2] = -1
    classes[3, 1] = classes[3, 0]
    classes[4] = classes[4, 0]
    values[4] = values[4] - 2.0
    values[5, 2] = -INF
    values[6] = -INF
    values[7], classes[7] = values[7].flip(0), classes[7].flip(0)
    classes[8], values[8] = -1, -INF
    for row, certain in ((9, 0.0), (10, -1e-7), (11, -1e-4)):
        values[row] = -30.0
        values[row, 3] = certain
    values[12] = -50.0 if rest else values[12] + 500.0
    values[13] = torch.finfo(torch.float32).min
    values[14, 3], classes[14, 3] = math.nan, -1          # what an absent entry holds is not read
    classes[15, :5] = -1
    values[16, 2] = math.nan                              # what a present one holds is
    for dtype in DTYPES:
        for temperature in (1.0, 2.0):
            check(normal(n, K, seed=5, scale=2.0, dtype=dtype), values, classes, temperature, rest)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("K", [12, 64, 90, 1024, 1500])
@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16"])
def test_students_beyond_the_ordinary(K, rest, dtype):
    """Masks, rows of masks, far offsets, a rest of the student's that is far below its best classes, infinities and NaN."""
    n, k = 32, 5
    values, classes = teacher_of(n, K, k, rest, 1.0, 4)
    inside = torch.zeros(n, K, dtype=torch.bool, device="cuda").scatter_(1, classes.long(), True)
    x = normal(n, K, seed=6, scale=2.0)
    x[0] = -INF
    x[1] = torch.where(inside[1], x[1], -INF)             # no class is left outside the list
    x[2] = torch.where(inside[2], -INF, x[2])             # none in it
    x[3, classes[3, 1].long()] = -INF
    x[4] = torch.where(inside[4], x[4] + 60.0, x[4])      # a rest of 1e-26
    x[5] = torch.where(inside[5], x[5] + 200.0, x[5])     # below the smallest fp32
    x[6] = torch.where(inside[6], x[6] - 60.0, x[6])
    x[7] += 20000.0
    x[8] -= 20000.0
    x[9] = torch.finfo(dtype).min
    x[10, 1] = math.nan
    x[11, 2] = INF
    x[12] = 0.0
    x[13, ::2] = torch.finfo(dtype).min
    x[14] = torch.where(inside[14], x[14] + 40.0, x[14])  # about where the sum is taken again
    x[15] = torch.where(inside[15], x[15] + 46.0, x[15])
    check(x.to(dtype), values, classes, 1.0, rest)


@pytest.mark.parametrize("K", [30, 400, 3000])
def test_lists_that_hold_little(K):
    """Flat teachers and students: the list's share and the rest's differences are small beside 1, and lose nothing to it."""
    n = 64
    x, t = normal(n, K, seed=1) / 30, normal(n, K, seed=2) / 30
    out = F.class_log_probs(t, top=4)
    for a, b in ((out.top_log_probs, out.top_classes), (out.top_log_probs[:, :1], out.top_classes[:, :1])):
        check(x, a, b, rest=True)
        loss = F.distill_topk(x, a, b, rest=True)
        want = R.distill(x, a, b, 1.0, True, normal(n, seed=77))
        # the terms of a few hundredths of a flat list: a dozen roundings of the largest of them
        size = (a.double().exp() * (a.double() - torch.log_softmax(x.double(), 1).gather(1, b.long())).abs()).sum(1)
        assert ((loss.double() - want["loss"][0]).abs() <= 12 * 2.0 ** -22 * (size + a.double().exp().sum(1))).all()


@pytest.mark.parametrize("K", [20, 100, 1100])
def test_classes_out_of_range(K):
    values, classes = teacher_of(30, K, 4, False, 1.0)
    x = normal(30, K, seed=2)
    for wrong in (-2, K, K + 7, 2 ** 40, -2 ** 63):
        for dtype in (torch.int64, torch.int32):
            if dtype == torch.int32 and abs(wrong) > 2 ** 31:
                continue
            c = classes.to(dtype)
            c[11, 2] = wrong
            status = ops.new_status("cuda")
            out = check(x, values, c, status=status)
            assert int(status) == 1 and int(out.isnan().sum()) == 1
            with pytest.raises(_lib.Ptv3Error, match="out of range"):
                F.distill_topk(x, values, c)


@pytest.mark.parametrize("K", [20, 70, 1050])
def test_one_gradient_for_all_rows(K):
    values, classes = teacher_of(50, K, 4, True, 1.0)
    x = normal(50, K, seed=2).requires_grad_()
    got = torch.autograd.grad(F.distill_topk(x, values, classes, rest=True).mean(), x)[0]
    want = R.distill(x.detach(), values, classes, 1.0, True, torch.full((50,), 1 / 50, device="cuda"))
    R.assert_near(got, *want["dlogits"], "dlogits")
    g = normal(50, 3, seed=1)
    got = torch.autograd.grad(F.distill_topk(x, values, classes, rest=True), x, g[:, 1])[0]
    R.assert_near(got, *R.distill(x.detach(), values, classes, 1.0, True, g[:, 1])["dlogits"], "dlogits")


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16"])
def test_rows_of_wider_ones_and_other_strides(dtype):
    for n, K, first, width in ((130, 20, 3, 25), (65, 200, 8, 216), (65, 200, 1, 208), (9, 1200, 5, 1211), (1, 96, 7, 200)):
        wide = normal(n, width, seed=K, dtype=dtype)
        values, classes = teacher_of(n, K, 4, True, 1.0)
        check(wide[:, first:first + K], values, classes, rest=True)
    values, classes = teacher_of(33, 20, 8, True, 1.0)
    check(normal(20, 33, seed=1, dtype=dtype).t(), values[:, ::2], classes[:, ::2], rest=True)
    check(normal(1, 20, seed=1, dtype=dtype).expand(33, 20), values, classes, rest=True)


def test_rows_behind_four_gigabytes():
    n, K = 33000, 2 ** 17
    x = torch.zeros(n, K, device="cuda", dtype=torch.bfloat16)
    x[-3:] = normal(3, K, seed=1, dtype=torch.bfloat16)
    values, classes = torch.full((n, 3), -2.0, device="cuda"), torch.tensor([5, 9, K - 1], device="cuda").expand(n, 3)
    want = R.distill(x[-3:], values[-3:], classes[-3:], 1.0, True, torch.ones(3, device="cuda"))
    x.requires_grad_()
    loss = F.distill_topk(x, values, classes, rest=True)
    R.assert_near(loss[-3:], *want["loss"], "loss")
    dx = torch.autograd.grad(loss, x, torch.ones(n, device="cuda"))[0]
    R.assert_near(dx[-3:], *want["dlogits"], "dlogits")


@pytest.mark.parametrize("rest", [False, True])
def test_the_most_classes(rest):
    K = F.CLASSES_MAX
    check(normal(2, K, seed=9), *teacher_of(2, K, 64, rest, 1.0), rest=rest)


def test_no_points():
    x = torch.empty(0, 20, device="cuda", requires_grad=True)
    loss = F.distill_topk(x, torch.empty(0, 3, device="cuda"), torch.empty(0, 3, dtype=torch.int32, device="cuda"))
    assert loss.shape == (0,) and torch.autograd.grad(loss.sum(), x)[0].shape == (0, 20)


@pytest.mark.parametrize("K", [20, 200, 1500])
def test_other_streams_and_graphs(K):
    x = normal(300, K, seed=6, dtype=torch.bfloat16)
    values, classes = teacher_of(300, K, 8, True, 1.0)
    status, up = ops.new_status("cuda"), normal(300, seed=7)

    def step(x):
        leaf = x.detach().requires_grad_()
        loss = F.distill_topk(leaf, values, classes, rest=True, status=status)
        return [loss.detach(), torch.autograd.grad(loss, leaf, up)[0]]
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
            F.distill_topk(held, values, classes)
    assert int(status) == 0


def test_refusals():
    x = torch.zeros(4, 6, device="cuda")
    v, c = torch.zeros(4, 3, device="cuda"), torch.zeros(4, 3, dtype=torch.int32, device="cuda")
    for args, kw, word in (((x[0], v, c), {}, "logits"), ((x, v, c[:3]), {}, "classes"), ((x, v[:, :2], c), {}, "teacher"),
                           ((x, v, c.float()), {}, "classes"), ((x, v[:, :0], c[:, :0]), {}, "classes"), ((x, v, c[0]), {}, "classes"),
                           ((x, v.expand(4, 3), c), dict(temperature=0.0), "temperature"),
                           ((x, v.clone().requires_grad_(), c), {}, "detach"),
                           ((x, torch.zeros(4, 65, device="cuda"), torch.zeros(4, 65, dtype=torch.int32, device="cuda")), {}, "classes"),
                           ((x, v, c), dict(status=torch.zeros(1, device="cuda")), "status")):
        with pytest.raises(ValueError, match=word):
            F.distill_topk(*args, **kw)
    with pytest.raises(_lib.Ptv3Error, match="not supported"):
        F.distill_topk(x, v.half(), c)
    with pytest.raises(_lib.Ptv3Error, match="CUDA"):
        F.distill_topk(x, v, c.cpu())
    with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError):
        F.distill_topk(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)), v, c)


def test_a_teacher_scored_in_inference_mode():
    """What a scoring job leaves is what a student's step takes; the student that is the teacher has no loss and no gradient."""
    x = normal(200, 20, seed=1, scale=2.0)
    with torch.inference_mode():
        t = F.class_log_probs(x, top=6, temperature=2.0)
    leaf = x.clone().requires_grad_()
    loss = F.distill_topk(leaf, t.top_log_probs, t.top_classes, temperature=2.0, rest=True)
    dx = torch.autograd.grad(loss.sum(), leaf)[0]
    # t and p of a row of 20 classes are off by at most 40 roundings each, in a sum of seven logarithms of at most 20
    assert loss.abs().max() < 7 * 20 * 80 * 2.0 ** -24 and dx.abs().max() < 80 * 2.0 ** -24


@pytest.mark.parametrize("K", [20, 333, 1201])
def test_the_same_bits_on_every_run(K):
    x = normal(500, K, seed=6, dtype=torch.bfloat16)
    values, classes = teacher_of(500, K, 8, True, 1.0)

    def step():
        leaf = x.detach().requires_grad_()
        loss = F.distill_topk(leaf, values, classes, rest=True)
        return [loss, torch.autograd.grad(loss.sum(), leaf)[0]]
    first = step()
    assert all(torch.equal(a, b) for _ in range(3) for a, b in zip(first, step()))
