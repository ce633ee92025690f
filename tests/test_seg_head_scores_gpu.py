"""Scores straight from features against the formulas in 64 bits, the head that gives them, and a student that learns from its lists.

Features are multiples of 1/16, weights and biases of 1/256, small enough that every sum of products is exact in 32 bits: the logits are the
reference's, and the order of alternatives has one answer."""
import math

import pytest
import torch

import class_scores_reference as R
from pointtransformerv3_b200 import Point, SegHead, _lib, ops
from pointtransformerv3_b200 import functional as F

pytestmark = pytest.mark.gpu

INF = math.inf


def made(n, C, K, seed, bias=True):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")
    feat = ((normal(n, C) * 16).round() / 16).clamp(-4, 4).bfloat16()
    weight = ((normal(K, C) * (2 / math.sqrt(C)) * 256).round() / 256).clamp(-1, 1).bfloat16()
    b = ((normal(K) * 128).round() / 256).clamp(-0.5, 0.5).bfloat16() if bias else None
    return feat, weight, b


def labels_of(n, K, seed=0, dtype=torch.int64):
    return torch.randint(-1, K, (n,), generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def check(feat, weight, bias, labels=None, top=0, temperature=1.0, ignore_index=-1, status=None):
    own = status is None
    status = ops.new_status("cuda") if own else status
    got = ops.seg_head_log_probs(feat, weight, bias, labels, top, temperature, ignore_index, status)
    x = feat.double() @ weight.double().t()
    x = x if bias is None else x + bias.double()
    want = R.scores(x, labels, top, temperature, ignore_index)
    for name in ("log_prob", "entropy", "top_log_probs"):
        if name in want:
            R.assert_near(getattr(got, name), *want[name], name)
    if top:
        classes = torch.where(want["top_log_probs"][0] > -INF, want["top_classes"][0], -1)
        assert torch.equal(got.top_classes, classes), "top_classes"
    if own:
        assert int(status) == 0
    return got


@pytest.mark.parametrize("K", [1, 2, 7, 20, 32, 33, 64, 65, 100, 128, 129, 200, 256, 257, 300, 513, 1201, 2500])
def test_numbers_of_classes(K):
    for top in (0, 3, 8, 11, 16, 32):
        check(*made(300, 64, K, K + top), labels_of(300, K, K, torch.int32 if K % 2 else torch.int64), top, (1.0, 0.5, 3.0)[K % 3])


@pytest.mark.parametrize("C,K", [(8, 20000), (64, 20000), (512, 9001), (64, F.CLASSES_MAX)])
def test_long_lists_of_classes(C, K):
    for top in (0, 7, 16, 32):
        check(*made(70, C, K, top), labels_of(70, K), top)


@pytest.mark.parametrize("C", [8, 16, 24, 56, 64, 72, 96, 128, 200, 256, 264, 384, 448, 512])
def test_numbers_of_channels(C):
    for K, top in ((20, 5), (150, 8), (700, 16), (700, 2), (260, 0), (260, 32)):
        check(*made(200, C, K, C + K, bias=K != 150), labels_of(200, K), top)


@pytest.mark.parametrize("n", [1, 2, 31, 127, 128, 129, 1000, 128 * 148, 128 * 148 * 3 + 17])
def test_numbers_of_rows(n):
    for K, top in ((20, 4), (300, 8), (300, 12)):
        check(*made(n, 32, K, n), labels_of(n, K), top)


@pytest.mark.parametrize("top", list(range(1, 33)))
def test_numbers_of_alternatives(top):
    for K in (3, 40, 64, 90, 400):
        check(*made(150, 16, K, top), None, top)


@pytest.mark.parametrize("K", [20, 64, 130, 900])
def test_equal_logits_go_to_the_lowest_class(K):
    feat, weight, bias = made(140, 16, K, K)
    weight[:, 1:] = 0                            # a few values, many times
    bias = (torch.arange(K, device="cuda") % 3 / 2).bfloat16()
    feat[:9] = 0
    for top in (1, 8, 16, 32):
        check(feat, weight, bias, labels_of(140, K), top)
        check(feat, weight, torch.zeros_like(bias), labels_of(140, K), top)
    # rising and falling logits: each is better than all before it, or worse
    rising = torch.arange(K, device="cuda")
    rising = rising / 256 if K < 256 else rising // 8 / 128
    for bias in (rising, rising.flip(0)):
        check(torch.zeros_like(feat), weight, bias.bfloat16(), labels_of(140, K), 13)


@pytest.mark.parametrize("K", [20, 64, 100, 500, 1201])
def test_masked_classes_and_rows_that_are_no_numbers(K):
    feat, weight, bias = made(200, 64, K, K)
    bias[::2] = -INF
    bias[:min(40, K // 2)] = -INF                # a whole part of the row
    labels = labels_of(200, K)
    for top in (5, 16, 32):
        check(feat, weight, bias, labels, top)
    low = bias.clone()
    low[::2] = torch.finfo(torch.bfloat16).min
    check(feat, weight, low, labels, 4)
    bias[:] = -INF
    got = check(feat, weight, bias, labels, 5)
    assert (got.entropy == 0).all() and (got.top_classes == -1).all()
    # NaN and plus infinity: the rows that hold one, no others
    feat, weight, bias = made(200, 64, K, K)
    clean = ops.seg_head_log_probs(feat, weight, bias, labels, 5)
    feat[17, 3], feat[140, 5] = math.nan, INF
    got = ops.seg_head_log_probs(feat, weight, bias, labels, 5)
    hit = torch.zeros(200, dtype=torch.bool, device="cuda")
    hit[17] = hit[140] = True
    assert got.entropy[hit].isnan().all() and got.top_log_probs[hit].isnan().all() and (got.top_classes[hit] == -1).all()
    for a, b in zip(got, clean):
        assert torch.equal(a[~hit], b[~hit])


def test_labels_out_of_range():
    feat, weight, bias = made(150, 64, 200, 1)
    for wrong in (-1, -2, 200, 2 ** 40, -2 ** 63):
        labels = torch.zeros(150, dtype=torch.int64, device="cuda")
        labels[140] = wrong
        status = ops.new_status("cuda")
        got = check(feat, weight, bias, labels, 3, ignore_index=-100, status=status)
        assert int(status) == 1 and got.log_prob[140].isnan()
        with pytest.raises(_lib.Ptv3Error, match="out of range"):
            ops.seg_head_log_probs(feat, weight, bias, labels, ignore_index=-100)


def test_ordinary_features():
    """Values as layers give them: a logit is off by at most 2^-22 for each product of 16 of the sum of its products' sizes, a log probability by
    twice that."""
    g = torch.Generator(device="cuda").manual_seed(1)
    for C, K in ((64, 20), (512, 700)):
        feat = torch.randn(400, C, generator=g, device="cuda").bfloat16()
        weight = (torch.randn(K, C, generator=g, device="cuda") / 8).bfloat16()
        labels = torch.randint(0, K, (400,), generator=g, device="cuda")
        got = ops.seg_head_log_probs(feat, weight, None, labels, 4)
        want = R.scores(feat.double() @ weight.double().t(), labels, 4)
        off = (feat.double().abs() @ weight.double().abs().t()).amax(1) * (C / 16 + 2) * 2.0 ** -22
        R.assert_near(got.log_prob, want["log_prob"][0], want["log_prob"][1] + 2 * off)
        R.assert_near(got.top_log_probs, want["top_log_probs"][0], want["top_log_probs"][1] + 2 * off[:, None])


@pytest.mark.parametrize("C,K,top", [(64, 20, 4), (96, 500, 9)])
def test_other_streams_graphs_and_runs(C, K, top):
    feat, weight, bias = made(5000, C, K, 1)
    labels, status = labels_of(5000, K), ops.new_status("cuda")

    def call(f):
        return ops.seg_head_log_probs(f, weight, bias, labels, top, status=status)
    want = call(feat)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(call(feat), want))
    sides = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for side in sides:                           # two calls at once
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got.append(call(feat))
    for side in sides:
        torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
    held = feat.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call(held)
    held.copy_(made(5000, C, K, 2)[0])
    want = call(held)
    graph.replay()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and int(status) == 0


def test_layouts():
    """Slices and other orders are copied, empty batches answered."""
    feat, weight, bias = made(100, 64, 30, 1)
    want = ops.seg_head_log_probs(feat, weight, bias, top=3)
    wide = torch.zeros(100, 71, device="cuda", dtype=torch.bfloat16)
    wide[:, 5:69] = feat
    for f, w, b in ((wide[:, 5:69], weight, bias), (feat.t().contiguous().t(), weight, bias), (feat, torch.cat([bias[:1], weight.flatten()])[1:].view(30, 64), bias),
                    (feat, weight, torch.cat([bias[:1], bias])[1:])):
        assert all(a is b or torch.equal(a, b) for a, b in zip(ops.seg_head_log_probs(f, w, b, top=3), want))
    empty = ops.seg_head_log_probs(feat[:0], weight, bias, torch.empty(0, dtype=torch.int64, device="cuda"), 3)
    assert empty.log_prob.shape == (0,) and empty.top_classes.shape == (0, 3)


def test_refusals():
    feat, weight, bias = made(10, 64, 30, 1)
    lab = torch.zeros(10, dtype=torch.int64, device="cuda")
    for args, kw, word in (((feat[0], weight, bias), {}, "features"), ((feat, weight[:, :32], bias), {}, "features"), ((feat, weight[:0], None), {}, "classes"),
                           ((feat, weight, bias[:5]), {}, "bias"), ((feat.float(), weight, bias), {}, "bf16"), ((feat, weight, bias.float()), {}, "bf16"),
                           ((feat, weight, bias, lab[:4]), {}, "labels"), ((feat, weight, bias), dict(top=33), "alternatives"),
                           ((feat, weight, bias), dict(top=65), "alternatives"), ((feat, weight, bias), dict(temperature=0.0), "temperature"),
                           ((feat[:, :60].contiguous(), weight[:, :60].contiguous(), bias), {}, "channels")):
        with pytest.raises(ValueError, match=word):
            ops.seg_head_log_probs(*args, **kw)
    with pytest.raises(_lib.Ptv3Error, match="CUDA"):
        ops.seg_head_log_probs(feat, weight.cpu(), bias)
    for t in (feat, weight, bias):
        t.requires_grad_()
        with pytest.raises(ValueError, match="gradients"):
            ops.seg_head_log_probs(feat, weight, bias)
        with torch.no_grad():
            assert not ops.seg_head_log_probs(feat, weight, bias).entropy.requires_grad
        t.requires_grad_(False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_head_scores_its_own_logits(dtype):
    """SegHead.log_probs: from features where nothing asks for gradients, else from the layer's logits; of a Point as of a matrix."""
    torch.manual_seed(0)
    head = SegHead(64, 20).cuda().to(dtype)
    feat = torch.randn(500, 64, device="cuda").to(dtype)
    labels = labels_of(500, 20)
    with torch.no_grad():
        plain = head.log_probs(feat, labels, top=5)
        point = Point(feat=feat, coord=torch.rand(500, 3, device="cuda"), offset=torch.tensor([500], device="cuda"))
        of_point = head.log_probs(point, labels, top=5)
    assert all(torch.equal(a, b) for a, b in zip(plain, of_point))
    feat = feat.clone().requires_grad_()
    out = head.log_probs(feat, labels, top=5)
    # the layer's logits are rounded to its type (up to 8 in size here), those on the way to the scores are not
    step = 8 * torch.finfo(dtype).eps + 64 * 2.0 ** -22
    assert (out.log_prob - plain.log_prob).abs().max() < 2 * step and (out.entropy - plain.entropy).abs().max() < 10 * step
    grads = torch.autograd.grad(-out.log_prob.mean(), [feat, head.linear.weight, head.linear.bias])
    # the same gradients by torch's own operators, in 64 bits from the same logits
    leaves = [t.detach().double().requires_grad_() for t in (feat, head.linear.weight, head.linear.bias)]
    loss = torch.nn.functional.cross_entropy(torch.nn.functional.linear(*leaves), labels, ignore_index=-1, reduction="sum") / 500
    for got, want in zip(grads, torch.autograd.grad(loss, leaves)):
        assert (got.double() - want).norm() <= want.norm() * 8 * torch.finfo(dtype).eps + 1e-7


def test_a_student_learns_from_a_teachers_head():
    """A teacher's head scores a batch, its lists are what a student's step takes: a loss for every point, gradients of every weight."""
    torch.manual_seed(0)
    teacher, student = SegHead(64, 40).cuda().bfloat16(), SegHead(32, 40).cuda().bfloat16()
    feats = torch.randn(1000, 64, device="cuda").bfloat16(), torch.randn(1000, 32, device="cuda").bfloat16()
    status = ops.new_status("cuda")
    with torch.inference_mode():
        lists = teacher.log_probs(feats[0], top=8, temperature=2.0, status=status)
    labels = labels_of(1000, 40)
    logits = student.linear(feats[1])
    kept = R.distill(logits.detach(), lists.top_log_probs, lists.top_classes, 2.0, True)
    loss = F.distill_topk(logits, lists.top_log_probs, lists.top_classes, temperature=2.0, rest=True, status=status)
    R.assert_near(loss, *kept["loss"], "loss")
    hard = F.class_log_probs(logits, labels, status=status)
    (4.0 * loss.mean() - hard.log_prob.sum() / (labels >= 0).sum()).backward()
    assert all(p.grad is not None and p.grad.abs().sum() > 0 for p in student.parameters())
    assert int(status) == 0
