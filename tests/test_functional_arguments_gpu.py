"""Arguments of the trainable operators as programs have them: slices of larger buffers, tensors that change, other modes of torch."""
import pytest
import torch

import functional_norms as N
import functional_reference as R
from pointtransformerv3_b200 import _lib, ops
from pointtransformerv3_b200 import functional as F

pytestmark = pytest.mark.gpu


def normal(*shape, seed, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("D", [8, 16, 64, 128])
def test_weights_from_a_buffer_of_parameters(D, dtype):
    """Norm weights that are slices of one buffer, behind an odd number of values: the same bits as copies of them, forward and
    in all gradients."""
    n, heads = 77, 2
    qkv = normal(n, 3 * heads * D, seed=1, dtype=dtype)
    dout = normal(n, 3 * heads * D, seed=2, dtype=dtype)
    buffer = 1 + normal(2 * D + 9, seed=3, dtype=dtype, scale=0.2)
    grid = torch.randint(0, 99, (n, 3), generator=torch.Generator().manual_seed(4), dtype=torch.int32).cuda()

    def run(q, k):
        x, q, k = (t.detach().requires_grad_() for t in (qkv, q, k))
        out = F.qk_norm_rope(x, heads, grid, q, k)
        return (out,) + torch.autograd.grad(out, (x, q, k), dout)
    for first in (0, 1, 2, 3, 5):
        q, k = buffer[first:first + D], buffer[first + D + 1:first + 2 * D + 1]
        assert (q.data_ptr() - buffer.data_ptr()) == first * buffer.element_size()
        assert all(torch.equal(a, b) for a, b in zip(run(q, k), run(q.clone(), k.clone())))


def patches(counts, patch, seed=0, extent=12):
    """A batch of scenes in random order, their patches and coordinates."""
    g = torch.Generator().manual_seed(seed)
    order, at = [], 0
    for c in counts:
        order.append(torch.randperm(c, generator=g) + at)
        at += c
    pad, unpad, cu = ops.pad_plan(torch.cumsum(torch.tensor(counts), 0).cuda(), counts, patch)
    grid = torch.randint(0, extent, (at, 3), generator=g, dtype=torch.int32).cuda()
    return dict(n=at, geometry=(torch.cat(order).cuda(), pad, unpad, cu), grid=grid, longest=min(max(counts), patch))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_index_tensors_of_inference_mode_are_kept_as_they_were(dtype):
    """They count no changes, so a gradient has a copy of them: it is the one of the forward pass's coordinates, buckets and
    sequences, whatever they hold by then."""
    p = patches([150, 60], 64)
    H, C = 2, 32
    with torch.inference_mode():
        grid, cu = p["grid"].clone(), p["geometry"][3].clone()
        buckets, num = F.log_buckets(10)
        buckets = buckets.cuda()
    qkv = normal(p["n"], 3 * C, seed=1, dtype=dtype).requires_grad_()
    table, w = normal(3 * num, H, seed=2).requires_grad_(), torch.ones(C // H, device="cuda")
    dout = normal(p["n"], C, seed=3, dtype=dtype)
    args = p["geometry"][:3] + (cu, H, p["longest"])
    outs = [F.attention_bias(qkv, *args, grid_coord=grid, table=table, buckets=buckets),
            F.qk_norm_rope(qkv, H, grid, w, w)]

    def grads():
        return (torch.autograd.grad(outs[0], (qkv, table), dout, retain_graph=True)
                + torch.autograd.grad(outs[1], qkv, qkv.detach(), retain_graph=True))
    first = grads()
    with torch.inference_mode():
        grid.mul_(300)
        buckets.zero_()
        cu.zero_()
    assert all(torch.equal(a, b) for a, b in zip(first, grads()))


@pytest.mark.parametrize("width", [16, 32, 64])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_coordinates_that_change_unseen_stay_in_the_table(width, dtype):
    """Written behind torch's back, coordinates make a gradient of nothing in particular; it reads and writes what it owns, and with the
    coordinates back it is what it was."""
    p = patches([300, 77], 128)
    qkv = normal(p["n"], 3 * 2 * width, seed=1, dtype=dtype).requires_grad_()
    table, dout = normal(3 * 63, 2, seed=2).requires_grad_(), normal(p["n"], 2 * width, seed=3, dtype=dtype)
    out = F.attention_bias(qkv, *p["geometry"], 2, p["longest"], grid_coord=p["grid"], table=table)

    def grads():
        return torch.autograd.grad(out, (qkv, table), dout, retain_graph=True)
    first, grid = grads(), p["grid"].clone()
    for change in (lambda g: g * 1000 - 7, lambda g: g - 2 ** 31, lambda g: 2 ** 31 - 1 - g):
        p["grid"].data.copy_(change(grid.long()).clamp(-2 ** 31, 2 ** 31 - 1))
        assert all(bool(t.isfinite().all()) for t in grads())
    p["grid"].data.copy_(grid)
    assert all(torch.equal(a, b) for a, b in zip(first, grads()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("counts,patch", [([17] * 200 + [1500], 1024), ([1] * 300 + [700, 2], 512), ([600] + [33] * 90, 300)],
                         ids=["17s", "1s", "33s"])
def test_short_sequences_beside_a_long_one(counts, patch, dtype):
    """Blocks of keys numbered by rows: results, gradients and the table's, and sequences of no rows among them."""
    p = patches(counts, patch)
    order, pad, unpad, cu = p["geometry"]
    ends = cu.tolist()
    cu = torch.tensor(ends[:1] * 3 + ends[1:40] + ends[39:40] * 2 + ends[40:] + ends[-1:], dtype=torch.int32, device="cuda")
    for width, H in ((16, 2), (64, 1)):
        C = width * H
        qkv, dout = normal(p["n"], 3 * C, seed=1, dtype=dtype), normal(p["n"], C, seed=3, dtype=dtype)
        buckets, num = F.log_buckets(130, device="cuda")
        x, table = qkv.clone().requires_grad_(), normal(3 * num, H, seed=2, scale=0.5).requires_grad_()
        out = F.attention_bias(x, order, pad, unpad, cu, H, p["longest"], grid_coord=p["grid"], table=table, buckets=buckets)
        got = (out,) + torch.autograd.grad(out, (x, table), dout)
        ref = R.attention(qkv, order, pad, unpad, cu, H, width ** -0.5, 1, table.detach(), p["grid"], 130, buckets, dout)
        for name, t in zip(("out", "dqkv", "dparam"), got):
            N.check(t.detach(), ref, name, qkv, dout, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_an_order_that_holds_a_point_twice_is_reported(dtype):
    """Another point has no row then, and nothing would write its result: in heads alone and together, in the first patch, in the last
    one and across two, with a graph and without one."""
    p = patches([130, 90, 1], 64)
    for width, H in ((16, 1), (32, 2), (64, 1)):
        qkv = normal(p["n"], 3 * width * H, seed=1, dtype=dtype)
        lam, rest = torch.ones(H, device="cuda"), p["geometry"][1:]
        for at, instead in ((3, 4), (0, 129), (200, 70), (219, 131)):
            order = p["geometry"][0].clone()
            order[at] = order[instead]
            for x in (qkv, qkv.clone().requires_grad_()):
                with pytest.raises(_lib.Ptv3Error, match="index or size out of range"):
                    F.attention_diff(x, lam, order, *rest, H, 64)
                with pytest.raises(_lib.Ptv3Error, match="index or size out of range"):
                    F.attention_bias(x, order, *rest, H, 64, grid_coord=p["grid"], table=torch.ones(9, H, device="cuda"))
        F.attention_diff(qkv, lam, *p["geometry"], H, 64)
