"""Trainable operators of serialized attention against their plain forms in 64 bits (functional_reference.py)."""
import math

import pytest
import torch

import functional_reference as R
from pointtransformerv3_b200 import _lib, ops
from pointtransformerv3_b200 import functional as F

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]
IDS = ["fp32", "bf16"]


def plan(counts, patch, seed=0, extent=12, spread=None):
    """A batch of scenes: random point order, patches of ops.pad_plan, coordinates."""
    g = torch.Generator().manual_seed(seed)
    n = sum(counts)
    order, at = [], 0
    for c in counts:
        order.append(torch.randperm(c, generator=g) + at)
        at += c
    offset = torch.cumsum(torch.tensor(counts), 0).cuda()
    pad, unpad, cu = ops.pad_plan(offset, counts, patch)
    grid = torch.randint(0, extent, (n, 3), generator=g, dtype=torch.int32)
    return dict(order=torch.cat(order).cuda(), pad=pad, unpad=unpad, cu=cu, grid=grid.cuda(), n=n,
                longest=min(max(counts), patch))


def normal(*shape, seed, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def geometry(p):
    return p["order"], p["pad"], p["unpad"], p["cu"]


# scenes, patch: one point; short of a patch; whole patches; a borrowed tail of one row and of nearly all; many short ones; odd
PLANS = [([1], 16), ([5], 64), ([64, 128], 64), ([65], 64), ([1, 127, 3], 64), ([17] * 9, 48), ([333, 200], 111), ([1024], 1024),
         ([1500], 1024), ([70, 1, 900], 257)]


def run_bias(p, C, H, dtype, table_dtype, bound, buckets=None, num=None, seed=1, offset=0.0, scale=None, table_scale=0.5):
    qkv = normal(p["n"], 3 * C, seed=seed)
    qkv[:, 2 * C:] += offset
    qkv = qkv.to(dtype).requires_grad_()
    num = num or 2 * bound + 1
    table = normal(3 * num, H, seed=seed + 1, dtype=table_dtype, scale=table_scale).requires_grad_()
    dout = normal(p["n"], C, seed=seed + 2, dtype=dtype)
    out = F.attention_bias(qkv, *geometry(p), H, p["longest"], scale, grid_coord=p["grid"], table=table, buckets=buckets)
    dqkv, dtable = torch.autograd.grad(out, (qkv, table), dout)
    ref = R.attention(qkv.detach(), *geometry(p), H, scale or (C // H) ** -0.5, 1, table.detach(), p["grid"], bound, buckets,
                      dout)
    return out, dqkv, dtable, ref


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("counts,patch", PLANS, ids=lambda v: str(v)[:20])
def test_bias_matches_64_bits(counts, patch, dtype):
    p = plan(counts, patch)
    for width, H in ((16, 3), (32, 1), (64, 2)):
        out, dqkv, dtable, ref = run_bias(p, width * H, H, dtype, dtype, 7)
        for name, got in (("out", out), ("dqkv", dqkv), ("dparam", dtable)):
            R.check(got, ref, name, width, p["longest"], dtype, "width %d" % width)


@pytest.mark.parametrize("bound,log", [(0, False), (1, False), (31, False), (64, False), (65, False), (130, True),
                                       (200, False), (512, True)])
@pytest.mark.parametrize("dtype,table_dtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                               (torch.bfloat16, torch.bfloat16)])
def test_bias_buckets(bound, log, dtype, table_dtype):
    p = plan([300, 450], 256, extent=max(4, 2 * bound))
    buckets, num = F.log_buckets(bound, device="cuda") if log else (None, None)
    out, dqkv, dtable, ref = run_bias(p, 32, 2, dtype, table_dtype, bound, buckets, num)
    for name, got in (("out", out), ("dqkv", dqkv), ("dparam", dtable)):
        R.check(got, ref, name, 16, p["longest"], dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_values_with_a_large_mean(dtype):
    """Values far from zero: the gradient of a score is the small difference of large numbers."""
    p = plan([400, 70], 256)
    out, dqkv, dtable, ref = run_bias(p, 32, 2, dtype, dtype, 9, offset=20.0)
    for name, got in (("out", out), ("dqkv", dqkv), ("dparam", dtable)):
        R.check(got, ref, name, 16, p["longest"], dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("counts,patch", PLANS, ids=lambda v: str(v)[:20])
def test_plain_attention_matches_64_bits(counts, patch, dtype):
    p = plan(counts, patch)
    for width, H in ((16, 2), (32, 1), (64, 1)):
        C = width * H
        qkv = normal(p["n"], 3 * C, seed=3, dtype=dtype).requires_grad_()
        dout = normal(p["n"], C, seed=4, dtype=dtype)
        out = F.attention_bias(qkv, *geometry(p), H, p["longest"])
        dqkv, = torch.autograd.grad(out, qkv, dout)
        ref = R.attention(qkv.detach(), *geometry(p), H, width ** -0.5, dout=dout)
        R.check(out, ref, "out", width, p["longest"], dtype)
        R.check(dqkv, ref, "dqkv", width, p["longest"], dtype)


def run_diff(p, C, H, dtype, lam_dtype, seed=5, lam=None, offset=0.0, size=1.0):
    qkv = normal(p["n"], 3 * C, seed=seed, scale=size)
    qkv[:, 2 * C:] += offset
    qkv = qkv.to(dtype).requires_grad_()
    lam = (torch.linspace(-0.3, 1.1, H) if lam is None else torch.full((H,), lam)).to(lam_dtype).cuda().requires_grad_()
    dout = normal(p["n"], C, seed=seed + 1, dtype=dtype)
    out = F.attention_diff(qkv, lam, *geometry(p), H, p["longest"])
    dqkv, dlam = torch.autograd.grad(out, (qkv, lam), dout)
    ref = R.attention(qkv.detach(), *geometry(p), H, (C // H // 2) ** -0.5, 2, lam.detach(), dout=dout)
    return out, dqkv, dlam, ref


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("counts,patch", PLANS, ids=lambda v: str(v)[:20])
def test_diff_matches_64_bits(counts, patch, dtype):
    p = plan(counts, patch)
    for width, H, lam_dtype in ((16, 3, torch.float32), (32, 1, dtype), (64, 2, dtype)):
        out, dqkv, dlam, ref = run_diff(p, width * H, H, dtype, lam_dtype)
        for name, got in (("out", out), ("dqkv", dqkv), ("dparam", dlam)):
            R.check(got, ref, name, width, p["longest"], dtype, "width %d" % width)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("lam,offset,size", [(0.0, 0.0, 1.0), (1.0, 8.0, 1.0), (0.8, 0.0, 6.0)])
def test_diff_weights_and_peaks(dtype, lam, offset, size):
    """No second map, values with a mean that the maps take from each other, and scores so large that a row is one key."""
    p = plan([500, 90], 256)
    out, dqkv, dlam, ref = run_diff(p, 64, 2, dtype, torch.float32, lam=lam, offset=offset, size=size)
    for name, got in (("out", out), ("dqkv", dqkv), ("dparam", dlam)):
        R.check(got, ref, name, 32, p["longest"], dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("scale", [-0.3, 0.01, 1.7])
def test_scales(dtype, scale):
    p = plan([150, 40], 64)
    out, dqkv, dtable, ref = run_bias(p, 32, 2, dtype, dtype, 5, scale=scale)
    for name, got in (("out", out), ("dqkv", dqkv), ("dparam", dtable)):
        R.check(got, ref, name, 16, p["longest"], dtype)
    qkv, lam = normal(190, 192, seed=1, dtype=dtype).requires_grad_(), torch.tensor([0.6], device="cuda", requires_grad=True)
    dout = normal(190, 64, seed=2, dtype=dtype)
    out = F.attention_diff(qkv, lam, *geometry(p), 1, 64, scale)
    dqkv, dlam = torch.autograd.grad(out, (qkv, lam), dout)
    ref = R.attention(qkv.detach(), *geometry(p), 1, scale, 2, lam.detach(), dout=dout)
    for name, got in (("out", out), ("dqkv", dqkv), ("dparam", dlam)):
        R.check(got, ref, name, 64, p["longest"], dtype)


def test_a_learned_table_follows_far_and_uneven_patches():
    """Patches whose points lie within a few cells beside ones that span thousands, and a table for offsets up to 512."""
    p = plan([256, 256, 300], 256)
    p["grid"][256:512] *= 400
    p["grid"][512:] *= 45
    for dtype in DTYPES:
        out, dqkv, dtable, ref = run_bias(p, 32, 2, dtype, dtype, 512)
        for name, got in (("out", out), ("dqkv", dqkv), ("dparam", dtable)):
            R.check(got, ref, name, 16, p["longest"], dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_buckets_that_mask(dtype):
    """Entries of minus infinity take keys out of a row, entries of the type's lowest value do the same, and a row that they leave
    without a key is NaN, as softmax has it; the others keep their values and gradients."""
    p = plan([256, 300], 128, extent=9)
    C, H, bound = 32, 2, 5
    qkv = normal(p["n"], 3 * C, seed=1, dtype=dtype)
    table = normal(3 * (2 * bound + 1), H, seed=2, dtype=dtype, scale=0.5)
    for low in (float("-inf"), torch.finfo(dtype).min):
        masked = table.clone()
        masked[[0, 1, 9, 13, 31], :] = low                 # (offsets of zero, which every row has with itself, stay)
        x, w = qkv.clone().requires_grad_(), masked.clone().requires_grad_()
        dout = normal(p["n"], C, seed=3, dtype=dtype)
        out = F.attention_bias(x, *geometry(p), H, p["longest"], grid_coord=p["grid"], table=w)
        got = (out,) + torch.autograd.grad(out, (x, w), dout)
        minus = torch.where(masked < -1e30, torch.full_like(masked, float("-inf")), masked)
        ref = R.attention(qkv, *geometry(p), H, 0.25, 1, minus, p["grid"], bound, None, dout)
        for name, t in zip(("out", "dqkv", "dparam"), got):
            R.check(t, ref, name, 16, p["longest"], dtype, name)
    nothing = torch.full_like(table, float("-inf"))
    out = F.attention_bias(qkv, *geometry(p), H, p["longest"], grid_coord=p["grid"], table=nothing)
    assert bool(out.isnan().all())


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_ordered_points(dtype):
    """Points along a curve, whose neighbours in the order share coordinates, and ones that all share them."""
    g = torch.arange(700)
    for grid in (torch.stack([g // 64, g // 8 % 8, g % 8], 1), torch.stack([g // 350, g * 0 + 3, g * 0 - 5], 1),
                 torch.stack([g, -g, g % 9], 1)):
        p = plan([700], 256)
        p["order"] = torch.arange(700, device="cuda")
        p["grid"] = grid.int().cuda()
        out, dqkv, dtable, ref = run_bias(p, 32, 2, dtype, dtype, 31)
        for name, got in (("out", out), ("dqkv", dqkv), ("dparam", dtable)):
            R.check(got, ref, name, 16, p["longest"], dtype)


# --------------------------------------------------------------------------- norms and rotation
def run_qk(n, heads, D, dtype, weight_dtype, norm, rope, extent=65536, seed=7):
    qkv = normal(n, 3 * heads * D, seed=seed, dtype=dtype).requires_grad_()
    ws = [(1 + normal(D, seed=seed + i, scale=0.2)).to(weight_dtype).requires_grad_() for i in (1, 2)] if norm else [None] * 2
    g = torch.Generator().manual_seed(seed)
    grid = torch.randint(-extent, extent, (n, 3), generator=g, dtype=torch.int32).cuda() if rope else None
    out = F.qk_norm_rope(qkv, heads, grid, *ws)
    dout = normal(n, 3 * heads * D, seed=seed + 3, dtype=dtype)
    leaves = [qkv] + (ws if norm else [])
    got = (out,) + torch.autograd.grad(out, leaves, dout)
    # the same in 64 bits
    wide = [t.detach().double().requires_grad_() for t in leaves]
    ref = R.qk_norm_rope(wide[0], heads, grid, *(wide[1:] if norm else (None, None)))
    return got, (ref,) + torch.autograd.grad(ref, wide, dout.double())


@pytest.mark.parametrize("dtype,weight_dtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                                (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("n,heads,D", [(1, 1, 8), (7, 3, 16), (341, 1, 8), (1000, 4, 16), (129, 2, 32), (65, 2, 64), (33, 1, 128),
                                       (5, 64, 16), (2, 40, 64), (20011, 2, 16)])
@pytest.mark.parametrize("norm,rope", [(True, True), (True, False), (False, True)])
def test_qk_norm_rope_matches_64_bits(n, heads, D, dtype, weight_dtype, norm, rope):
    (out, dqkv, *dws), (ref, dref, *dwref) = run_qk(n, heads, D, dtype, weight_dtype, norm, rope)
    half, e32 = R.HALF_STEP[dtype], 2.0 ** -24
    # a row's sum of squares, its root, the weight, cos and sin (2^-22 with the angle's), two products: of a head's size
    eps = (D + 16) * e32 + 2.0 ** -21
    for got, want in ((out, ref), (dqkv, dref)):
        size = want.reshape(n, 3 * heads, D).norm(dim=-1, keepdim=True).expand(-1, -1, D).reshape(n, -1)
        if got is dqkv and norm:       # dx is what is left of dn after its part along x is taken out
            c = heads * D
            x = torch.cat([run_rows(n, heads, D, dtype)[:, :2 * c].reshape(n, 2 * heads, D).double().norm(dim=-1),
                           torch.full((n, heads), math.sqrt(D), dtype=torch.float64, device="cuda")], 1)
            dn = normal(n, 3 * c, seed=10, dtype=dtype).double().reshape(n, 3 * heads, D).norm(dim=-1) * 1.8
            size = size + (dn / (x / math.sqrt(D) + 1e-3))[..., None].expand(-1, -1, D).reshape(n, -1)
        tol = half * 1.01 * want.abs() + 4 * eps * size
        assert bool(((got.double() - want).abs() <= tol).all()), float(((got.double() - want).abs() / tol).max())
    for got, want in zip(dws, dwref):
        # a sum of n * heads terms of a size of about one, each off by eps, added in trees
        tol = R.HALF_STEP[weight_dtype] * 1.01 * want.abs() + n * heads * 4 * eps + 1e-6
        assert bool(((got.double() - want).abs() <= tol).all())


def run_rows(n, heads, D, dtype):
    return normal(n, 3 * heads * D, seed=7, dtype=dtype)


def test_rotation_depends_on_offsets_only_and_keeps_norms():
    """Rotated queries and keys have products that a common shift of all coordinates leaves alone, far from the origin too."""
    n, heads, D = 64, 2, 32
    qkv = normal(n, 3 * heads * D, seed=1)
    grid = torch.randint(0, 50, (n, 3), generator=torch.Generator().manual_seed(0), dtype=torch.int32).cuda()
    a, b = (F.qk_norm_rope(qkv, heads, grid + shift) for shift in (0, 1000000007))

    def products(x):
        q, k = (x[:, i * heads * D:(i + 1) * heads * D].reshape(n, heads, D).double() for i in (0, 1))
        return torch.einsum("ihd,jhd->hij", q, k)
    # each product of D terms of rotated values, off by 2^-21 of their size
    size = qkv[:, :2 * heads * D].reshape(n, 2 * heads, D).norm(dim=-1).max().double() ** 2
    assert float((products(a) - products(b)).abs().max()) <= 8 * 2.0 ** -21 * float(size)
    assert torch.equal(a[:, 2 * heads * D:], qkv[:, 2 * heads * D:])


# --------------------------------------------------------------------------- properties
def test_gradients_against_differences():
    """Along a direction, the slope of <out, dout> over a short way is the gradient's product with it (fp32: differences of
    bf16 results are rounding)."""
    p = plan([90, 33], 48)
    C, H, h = 32, 2, 2.0 ** -5
    qkv = normal(p["n"], 3 * C, seed=1).requires_grad_()
    table, lam = normal(3 * 11, H, seed=2).requires_grad_(), torch.tensor([0.4, 0.9], device="cuda", requires_grad=True)
    dout = normal(p["n"], C, seed=3)
    for f, param in ((lambda x, w: F.attention_bias(x, *geometry(p), H, 48, grid_coord=p["grid"], table=w), table),
                     (lambda x, w: F.attention_diff(x, w, *geometry(p), H, 48), lam)):
        for at, leaf in enumerate((qkv, param)):
            step = normal(*leaf.shape, seed=9) / math.sqrt(leaf.numel())
            args = [qkv.detach(), param.detach()]

            def along(t):
                moved = list(args)
                moved[at] = args[at] + t * step
                return float((f(*moved).double() * dout.double()).sum())
            # five points: the error of the slope is of fourth order in h
            slope = (8 * (along(h) - along(-h)) - (along(2 * h) - along(-2 * h))) / (12 * h)
            grad = torch.autograd.grad(f(qkv, param), (qkv, param), dout)[at]
            want = float((grad.double() * step.double()).sum())
            # results off by 2^-20 each, over the way h; and h^4 times a fifth derivative of the size of the first
            noise = 18 / 12 / h * 2.0 ** -20 * math.sqrt(p["n"] * C) * 4
            assert abs(slope - want) <= noise + 8 * h ** 4 * float(grad.double().norm() * step.double().norm()), (at, slope, want)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_same_bits_on_every_run(dtype):
    p = plan([700, 333], 256)
    first = None
    for _ in range(3):
        got = [t.detach().clone() for t in run_bias(p, 64, 4, dtype, dtype, 31)[:3] + run_diff(p, 64, 2, dtype, torch.float32)[:3]]
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


def test_a_poisoned_patch_stays_in_its_patch():
    """NaN and infinities of one patch reach its own rows and points that it lends, nobody else's."""
    p = plan([128, 64], 64)
    C, H = 32, 2
    for dtype in DTYPES:
        for value in (float("nan"), float("inf")):
            qkv = normal(p["n"], 3 * C, seed=1, dtype=dtype)
            clean = F.attention_bias(qkv, *geometry(p), H, 64, grid_coord=p["grid"], table=torch.ones(9, H, device="cuda"))
            bad = qkv.clone()
            bad[p["order"][70]] = value
            x = bad.clone().requires_grad_()
            out = F.attention_bias(x, *geometry(p), H, 64, grid_coord=p["grid"], table=torch.ones(9, H, device="cuda"))
            dx, = torch.autograd.grad(out, x, torch.ones_like(out))
            others = torch.cat([p["order"][:64], p["order"][128:]])
            assert torch.equal(out[others], clean[others])
            assert bool(torch.isfinite(dx[others]).all())
            assert bool(out[p["order"][64:128]].isnan().any())


def test_empty_batch_and_only_needed_gradients():
    z = torch.zeros(0, dtype=torch.int64, device="cuda")
    cu = torch.zeros(1, dtype=torch.int32, device="cuda")
    for dtype in DTYPES:
        qkv = torch.zeros(0, 96, dtype=dtype, device="cuda", requires_grad=True)
        table = torch.ones(9, 2, dtype=dtype, device="cuda", requires_grad=True)
        lam = torch.ones(2, device="cuda", requires_grad=True)
        for out, param in ((F.attention_bias(qkv, z, z, z, cu, 2, 16, grid_coord=torch.zeros(0, 3, dtype=torch.int32, device="cuda"),
                                             table=table), table),
                           (F.attention_diff(qkv, lam, z, z, z, cu, 2, 16), lam)):
            assert out.shape == (0, 32)
            dq, dp = torch.autograd.grad(out.sum(), (qkv, param))
            assert dq.shape == qkv.shape and not dp.any()
        w = torch.ones(16, dtype=dtype, device="cuda", requires_grad=True)
        out = F.qk_norm_rope(qkv, 2, None, w, w)
        assert not torch.autograd.grad(out.sum(), w)[0].any()
    p = plan([50], 32)
    qkv, table = normal(50, 96, seed=1), normal(9, 2, seed=2).requires_grad_()
    out = F.attention_bias(qkv, *geometry(p), 2, 32, grid_coord=p["grid"], table=table)
    assert torch.autograd.grad(out.sum(), table)[0].shape == (9, 2)
    with torch.no_grad():
        assert torch.equal(out, F.attention_bias(qkv, *geometry(p), 2, 32, grid_coord=p["grid"], table=table))


def test_sequences_of_no_rows_and_a_table_used_twice():
    """Patches of no rows between others, and one table in two calls, whose gradients add up."""
    p = plan([100, 30], 64)
    cu = p["cu"].tolist()
    cu = torch.tensor(cu[:1] + cu[:1] + cu[1:2] * 3 + cu[2:] + cu[-1:], dtype=torch.int32, device="cuda")
    for dtype in DTYPES:
        qkv, table = normal(130, 96, seed=1, dtype=dtype), normal(33, 2, seed=2, dtype=dtype).requires_grad_()
        dout = normal(130, 32, seed=3, dtype=dtype)

        def step(ends, times):
            out = sum(F.attention_bias(qkv, p["order"], p["pad"], p["unpad"], ends, 2, 64, grid_coord=p["grid"], table=table)
                      for _ in range(times))
            return out, torch.autograd.grad(out, table, dout)[0]
        (a, da), (b, db), (c, dc) = step(p["cu"], 1), step(cu, 1), step(p["cu"], 2)
        assert torch.equal(a, b) and torch.equal(da, db)
        assert torch.equal(dc, 2 * da) and torch.equal(c, 2 * a)


def test_strided_unaligned_and_other_stream():
    p = plan([150, 80], 64)
    n, C, H = p["n"], 32, 2
    lam = torch.tensor([0.5, 0.2], device="cuda")
    for dtype in DTYPES:
        qkv = normal(n, 3 * C, seed=1, dtype=dtype)
        want = F.attention_diff(qkv, lam, *geometry(p), H, 64)
        wide = torch.zeros(n, 3 * C + 5, dtype=dtype, device="cuda")
        wide[:, 3:3 + 3 * C] = qkv
        flat = torch.zeros(n * 3 * C + 1, dtype=dtype, device="cuda")
        flat[1:] = qkv.reshape(-1)
        for other in (wide[:, 3:3 + 3 * C], flat[1:].view(n, 3 * C), qkv.t().contiguous().t()):
            assert torch.equal(F.attention_diff(other, lam, *geometry(p), H, 64), want)
            assert torch.equal(F.qk_norm_rope(other, H, p["grid"]), F.qk_norm_rope(qkv, H, p["grid"]))
        # a gradient that comes in other strides
        x = qkv.clone().requires_grad_()
        g = normal(n, C, seed=2, dtype=dtype)
        a, = torch.autograd.grad(F.attention_diff(x, lam, *geometry(p), H, 64), x, g)
        b, = torch.autograd.grad(F.attention_diff(x, lam, *geometry(p), H, 64), x, g.t().contiguous().t())
        assert torch.equal(a, b)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            x2 = qkv.clone().requires_grad_()
            c, = torch.autograd.grad(F.attention_diff(x2, lam, *geometry(p), H, 64), x2, g)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(a, c)


def test_two_captured_steps_that_run_beside_each_other():
    """Forward and backward captured into two graphs, replayed on two streams with new inputs."""
    p = plan([600, 300], 256)
    C, H = 64, 4
    status = ops.new_status("cuda")
    leaves = [normal(p["n"], 3 * C, seed=i, dtype=torch.bfloat16).requires_grad_() for i in (1, 2)]
    table, dout = normal(3 * 13, H, seed=3).requires_grad_(), normal(p["n"], C, seed=4, dtype=torch.bfloat16)

    def step(x):
        w = torch.ones(16, dtype=torch.bfloat16, device="cuda")
        out = F.attention_bias(F.qk_norm_rope(x, H, p["grid"], w, w), *geometry(p), H, 256, grid_coord=p["grid"], table=table,
                               status=status)
        return (out,) + torch.autograd.grad(out, (x, table), dout)
    graphs, outs = [], []
    for x in leaves:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(x)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(x))
        graphs.append(g)
    with torch.no_grad():
        for i, x in enumerate(leaves):
            x.copy_(normal(p["n"], 3 * C, seed=20 + i, dtype=torch.bfloat16))
    streams = [torch.cuda.Stream() for _ in graphs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for x, got in zip(leaves, outs):
        assert all(torch.equal(a, b) for a, b in zip(got, step(x)))
    assert ops.read_status(status) == 0


def test_bad_plans_are_reported():
    """A plan that does not fit is told by the status word; what is read and written stays within the tensors."""
    p = plan([130, 20], 64)
    C, H = 32, 2
    qkv, lam = normal(150, 3 * C, seed=1).requires_grad_(), torch.ones(2, device="cuda")

    def bad(**change):
        q = dict(p, **change)
        with pytest.raises(_lib.Ptv3Error, match="index or size out of range"):
            F.attention_diff(qkv, lam, q["order"], q["pad"], q["unpad"], q["cu"], H, q["longest"])
        status = ops.new_status("cuda")
        out = F.attention_diff(qkv, lam, q["order"], q["pad"], q["unpad"], q["cu"], H, q["longest"], status=status)
        torch.autograd.grad(out, qkv, torch.ones_like(out))
        assert ops.read_status(status) == 1

    def changed(t, i, v):
        t = t.clone()
        t[i] = v
        return t
    for name, i, v in (("order", 5, 150), ("order", 5, -1), ("pad", 9, 150), ("pad", 9, -3), ("unpad", 0, 10 ** 12),
                       ("unpad", 0, -1), ("unpad", 3, 4), ("cu", 1, 3), ("cu", 1, -5), ("cu", 1, 10 ** 6), ("cu", 0, 1),
                       ("cu", -1, 100)):
        bad(**{name: changed(p[name], i, v)})
    bad(longest=63)
    # two rows borrowed from one point
    pad = p["pad"].clone()
    pad[140:142] = pad[100]
    bad(pad=pad)
    grid = p["grid"].clone()
    grid[17, 1] = 2 ** 22 + 1
    with pytest.raises(_lib.Ptv3Error, match="index or size out of range"):
        F.attention_bias(qkv, *geometry(p), H, 64, grid_coord=grid, table=torch.ones(9, H, device="cuda"))
    with pytest.raises(_lib.Ptv3Error, match="index or size out of range"):      # (not wrapped into 32 bits)
        F.attention_bias(qkv, *geometry(p), H, 64, grid_coord=p["grid"].long() + 2 ** 32, table=torch.ones(9, H, device="cuda"))
    buckets, num = F.log_buckets(12, device="cuda")
    buckets[3] = num
    with pytest.raises(_lib.Ptv3Error, match="index or size out of range"):
        F.attention_bias(qkv, *geometry(p), H, 64, grid_coord=p["grid"], table=torch.ones(3 * num, H, device="cuda"), buckets=buckets)
    # and a good one is good, with a patch size beyond all scenes too
    F.attention_diff(qkv, lam, *geometry(plan([130, 20], 2048)), H, 2048)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("counts,patch", [([700, 600], 256), ([900, 1, 399], 65), ([1300], 1024), ([420] * 3, 512)],
                         ids=lambda v: str(v)[:20])
def test_many_heads(counts, patch, dtype):
    """Launches with a block for more than half of the SMs, which are laid out differently from short ones."""
    p = plan(counts, patch)
    for width, H in ((16, 8), (32, 9)):
        for run in (lambda: run_bias(p, width * H, H, dtype, dtype, 9), lambda: run_diff(p, width * H, H, dtype, dtype)):
            out, dqkv, dparam, ref = run()
            for name, got in (("out", out), ("dqkv", dqkv), ("dparam", dparam)):
                R.check(got, ref, name, width, p["longest"], dtype, "width %d" % width)


def test_index_tensors_that_change_before_the_gradient():
    """A gradient of coordinates, buckets or sequences other than the forward pass's is refused, as autograd does for its own."""
    p = plan([100, 30], 64)
    H = 2
    qkv, table = normal(130, 96, seed=1).requires_grad_(), normal(33, H, seed=2).requires_grad_()
    buckets, num = F.log_buckets(12, device="cuda")
    wide = normal(3 * num, H, seed=3).requires_grad_()
    for name in ("grid", "cu", "buckets"):
        q = dict(p, grid=p["grid"].clone(), cu=p["cu"].clone(), buckets=buckets.clone())
        outs = [F.attention_bias(qkv, *geometry(q), H, 64, grid_coord=q["grid"], table=wide, buckets=q["buckets"])]
        if name == "grid":
            outs.append(F.qk_norm_rope(qkv, H, q["grid"]))
        q[name].add_(0)
        for out in outs:
            with pytest.raises(RuntimeError, match="modified in place"):
                torch.autograd.grad(out, qkv, torch.ones_like(out))
    out = F.attention_bias(qkv, *geometry(p), H, 2 ** 40, grid_coord=p["grid"], table=table)      # (a patch size beyond all)
    assert torch.equal(out, F.attention_bias(qkv, *geometry(p), H, 64, grid_coord=p["grid"], table=table))
    with torch.inference_mode():
        grid = p["grid"].clone()
    out = F.attention_bias(qkv, *geometry(p), H, 64, grid_coord=grid, table=table)
    torch.autograd.grad(out, qkv, torch.ones_like(out))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("width,H", [(16, 17), (32, 9)])
def test_long_launches(width, H, dtype):
    """Enough patches of more than 256 rows for blocks whose warps own two row tiles."""
    p = plan([3000, 1100], 512)
    for run in (lambda: run_bias(p, width * H, H, dtype, dtype, 9), lambda: run_diff(p, width * H, H, dtype, dtype)):
        out, dqkv, dparam, ref = run()
        for name, got in (("out", out), ("dqkv", dqkv), ("dparam", dparam)):
            R.check(got, ref, name, width, p["longest"], dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_long_launches_of_wide_heads(dtype):
    p = plan([1400, 800], 512)
    for H in (8, 11):
        out, dqkv, dtable, ref = run_bias(p, 64 * H, H, dtype, dtype, 9)
        for name, got in (("out", out), ("dqkv", dqkv), ("dparam", dtable)):
            R.check(got, ref, name, 64, p["longest"], dtype)
        with torch.no_grad():
            qkv, table = normal(p["n"], 192 * H, seed=1, dtype=dtype), normal(57, H, seed=2, dtype=dtype, scale=0.5)
            alone = F.attention_bias(qkv, *geometry(p), H, 512, grid_coord=p["grid"], table=table)
        assert torch.equal(alone, out)
