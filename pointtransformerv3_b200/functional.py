"""Operators of serialized attention that can be trained: functions of tensors with gradients.

``qk_norm_rope`` prepares the rows of a QKV projection (norms of queries and keys for each head, rotation by grid
coordinates), ``attention_bias`` and ``attention_diff`` are attention cores within the patches of a serialized order, with a
learned relative position bias by buckets or as the difference of two softmax maps.  They take the index tensors that
``ops.attention`` takes; ``SerializedAttention`` calls them for its options ``qk_norm``, ``enable_rope``, ``enable_rpe`` (in training, and
where its bias is by buckets or reaches beyond 64 cells) and ``differential``.

All of them run on the current stream of the tensors' device, keep nothing between calls, and can be captured into a graph (with a
``status`` word of the caller's: one that they make themselves is read at once, which waits for the device).  A backward pass
that is captured wants leaves which no eager graph holds at that time (``x.detach().requires_grad_()``): torch ties a leaf's
gradient to the stream of the graph that met it first.  Gradients are of first order and backward, and the same bits on every run;
tensors with a tangent of forward-mode differentiation are refused.
"""
import contextlib
import math

import torch
from torch.autograd import forward_ad

from . import _lib, ops

HEAD_WIDTHS = (16, 32, 64)    # of the attention operators
BUCKETS_MAX_BOUND = 512       # offsets beyond that many cells share the outermost bucket in any case


def log_buckets(bound, exact=8, per_octave=4, device=None):
    """Bucket of every offset -bound .. bound, as ``attention_bias`` takes them, and their number: offsets below ``exact`` cells
    have one each, then ``per_octave`` buckets to every doubling, each sign its own."""
    if not (1 <= bound <= BUCKETS_MAX_BOUND and exact >= 1 and per_octave >= 1):
        raise ValueError("bound in [1, %d], exact and per_octave from 1 on" % BUCKETS_MAX_BOUND)
    half = [d if d < exact else exact + int(math.log2(d / exact) * per_octave + 1e-9) for d in range(bound + 1)]
    rank = {b: i for i, b in enumerate(sorted(set(half)))}          # none is empty
    half = [rank[b] for b in half]
    lut = [half[-1] - b for b in half[:0:-1]] + [half[-1] + b for b in half]
    return torch.tensor(lut, dtype=torch.int32, device=device), 2 * half[-1] + 1


def _same_device(first, *others):
    _lib.require_cuda(first, *others)
    device = first.device
    for t in others:
        if t is not None and t.device != device:
            raise ValueError("tensors on %s and %s" % (device, t.device))


_HERE = contextlib.nullcontext()


def _on(device):
    """Makes the tensors' device the current one, where it is another (the guard costs as much as a launch)."""
    return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _no_tangents(*tensors):
    """Refuses tensors with a tangent: the kernels would return results without one, which torch takes as a derivative of zero."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("no forward-mode derivatives")


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _aligned(t):
    """Contiguous rows that start on 16 bytes, as the kernels read them."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _kept(t):
    """An index tensor as a backward pass keeps it.  One made in inference mode counts no changes, so it is copied."""
    return t.clone() if t is not None and t.is_inference() else t


def _versions(*tensors):
    """What autograd compares for the tensors that it keeps."""
    return [None if t is None else t._version for t in tensors]


def _unchanged(versions, *tensors):
    if _versions(*tensors) != versions:
        raise RuntimeError("coordinates, buckets or sequences that a gradient needs were modified in place since the forward pass")


def _check_qkv(qkv, heads):
    if qkv.dim() != 2 or qkv.shape[1] % 3 or heads < 1 or (qkv.shape[1] // 3) % heads:
        raise ValueError("qkv must be (N, 3C), C a multiple of %d heads: got %s" % (heads, tuple(qkv.shape)))
    _lib.dtype_id(qkv)


def _int32(t, shape, what):
    if tuple(t.shape) != shape or t.is_floating_point() or t.is_complex():
        raise ValueError("%s must be integers %s, got %s %s" % (what, shape, t.dtype, tuple(t.shape)))
    if t.dtype == torch.int64:        # beyond 32 bits: held at their ends, not wrapped into the range
        t = t.clamp(-2 ** 31, 2 ** 31 - 1)
    return t.to(torch.int32).contiguous()


# --------------------------------------------------------------------------- norms and rotation
class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, grid, q_weight, k_weight, heads, eps, base):
        out = ops.qk_norm_rope_fwd(qkv, heads, grid, q_weight, k_weight, eps, base)
        ctx.save_for_backward(qkv if q_weight is not None else None, q_weight, k_weight)
        grid = _kept(grid)
        ctx.args = grid, heads, eps, base
        ctx.versions = _versions(grid)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        qkv, q_weight, k_weight = ctx.saved_tensors
        grid, heads, eps, base = ctx.args
        _unchanged(ctx.versions, grid)
        with _on(dout.device):
            dqkv, dq, dk = ops.qk_norm_rope_bwd(qkv, _aligned(dout), heads, grid, q_weight, k_weight, eps, base)
        return dqkv, None, dq, dk, None, None, None


def qk_norm_rope(qkv, heads, grid_coord=None, q_weight=None, k_weight=None, eps=1e-6, base=100.0):
    """Queries and keys of a QKV matrix normalised and rotated, values as they are.

    qkv (N, 3C), split (3, heads, D).  With ``q_weight`` and ``k_weight`` (D,) every head's query and key is divided by its
    root mean square (``eps`` added to the mean square) and multiplied by the weight.  With ``grid_coord`` (N, 3) integers of 32 bits the
    pairs (2i, 2i+1), i < 3p, p = D // 6, are then turned by grid_coord[i // p] * base ** (-(i % p) / p), so that scores
    depend on the offset between two points; values beyond 6p are left.  D in 8, 16, 32, 64, 128; bf16 or fp32.  For
    ``attention_diff``, whose heads have two queries and two keys, pass twice its number of heads.  Returns a matrix like qkv."""
    _same_device(qkv, grid_coord, q_weight, k_weight)
    _no_tangents(qkv, q_weight, k_weight)
    _check_qkv(qkv, heads)
    D = qkv.shape[1] // 3 // heads
    if (q_weight is None) != (k_weight is None) or (q_weight is None and grid_coord is None):
        raise ValueError("weights of both queries and keys, coordinates, or all three")
    if q_weight is not None and (q_weight.shape != (D,) or k_weight.shape != (D,) or q_weight.dtype != k_weight.dtype):
        raise ValueError("weights must be (%d,) of one type" % D)
    if grid_coord is not None:
        grid_coord = _int32(grid_coord, (qkv.shape[0], 3), "grid_coord")
    qkv = _aligned(qkv)
    if q_weight is not None:
        q_weight, k_weight = q_weight.contiguous(), k_weight.contiguous()
    with _on(qkv.device):
        if not _wants_grad(qkv, q_weight, k_weight):
            return ops.qk_norm_rope_fwd(qkv, int(heads), grid_coord, q_weight, k_weight, float(eps), float(base))
        return _QkNormRope.apply(qkv, grid_coord, q_weight, k_weight, int(heads), float(eps), float(base))


# --------------------------------------------------------------------------- attention
class _PatchAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, param, plan, heads, max_seqlen, scale, maps, bias, status):
        out, rows, lse, second = ops.patch_attention_fwd(qkv, plan, heads, max_seqlen, scale, maps, param, bias, status, True)
        ctx.save_for_backward(qkv, param, out, lse, second)
        plan = plan[:3] + (_kept(plan[3]),)
        if bias is not None:
            bias = (_kept(bias[0]), _kept(bias[1])) + bias[2:]
        ctx.args = plan, heads, max_seqlen, scale, maps, bias, rows
        ctx.versions = _versions(plan[3], *(bias or ())[:2])
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        qkv, param, out, lse, second = ctx.saved_tensors
        plan, heads, max_seqlen, scale, maps, bias, rows = ctx.args
        _unchanged(ctx.versions, plan[3], *(bias or ())[:2])
        with _on(dout.device):
            dqkv, dparam = ops.patch_attention_bwd(qkv, plan, heads, max_seqlen, scale, maps, param, bias, out, rows, lse,
                                                   second, _aligned(dout), ctx.needs_input_grad[1])
        return (dqkv, dparam) + (None,) * 7


def _attend(qkv, param, order_row, pad, unpad, cu_seqlens, bias, heads, max_seqlen, scale, maps, status):
    _no_tangents(qkv, param)
    n, D = qkv.shape[0], qkv.shape[1] // 3 // heads
    if D not in HEAD_WIDTHS:
        raise ValueError("heads of %d values (supported: 16, 32, 64)" % D)
    if order_row.shape != (n,) or unpad.shape != (n,) or pad.dim() != 1 or not n <= pad.shape[0] <= 2 * n:
        raise ValueError("order_row and unpad must be (%d,), pad %d to %d rows" % (n, n, 2 * n))
    if cu_seqlens.dim() != 1 or cu_seqlens.dtype != torch.int32 or cu_seqlens.shape[0] < (2 if n else 1):
        raise ValueError("cu_seqlens must be a row of int32, the ends of one sequence and more")
    if any(t.dtype != torch.int64 for t in (order_row, pad, unpad)):
        raise ValueError("order_row, pad and unpad must be int64")
    if status is not None and (status.dtype != torch.int32 or status.numel() < 1):
        raise ValueError("status must be an int32 word")
    if int(max_seqlen) < 1:
        raise ValueError("max_seqlen %d" % max_seqlen)
    max_seqlen = min(int(max_seqlen), 2 ** 31 - 1)
    if scale is None:
        scale = (D // maps) ** -0.5
    if not (math.isfinite(scale) and scale):
        raise ValueError("scale %r" % scale)
    plan = tuple(t.contiguous() for t in (order_row, pad, unpad, cu_seqlens))
    qkv, param = _aligned(qkv), None if param is None else param.contiguous()
    own = status is None
    if own and torch.cuda.is_current_stream_capturing():
        raise ValueError("a captured call needs a status word of the caller's: one of its own is read at once")
    with _on(qkv.device):
        if own:
            status = ops.new_status(qkv.device)
        if _wants_grad(qkv, param):
            out = _PatchAttention.apply(qkv, param, plan, int(heads), max_seqlen, float(scale), maps, bias, status)
        else:
            out = ops.patch_attention_fwd(qkv, plan, int(heads), max_seqlen, float(scale), maps, param, bias, status)[0]
        if own:
            _lib.raise_on_status(status, "ptv3_patch_attention_fwd")
    return out


def attention_bias(qkv, order_row, pad, unpad, cu_seqlens, heads, max_seqlen, scale=None, grid_coord=None, table=None,
                   buckets=None, status=None):
    """Attention within patches with a learned relative position bias: (N, C).

    qkv (N, 3C), split (3, heads, D), D in 16, 32, 64, bf16 or fp32; order_row (N,), pad, unpad, cu_seqlens: one row of a serialized
    order and its patches (``ops.pad_plan``), of at most ``max_seqlen`` rows.  Scores are scale q.k (scale: D ** -0.5) plus
    the sum over the axes a of table[a * num + bucket(grid_coord[i, a] - grid_coord[j, a]), head]; table (3 num, heads), fp32 or
    bf16, grid_coord (N, 3) integers within 2^22 of zero.  ``buckets`` (2 bound + 1,) int32 gives the bucket of every offset -bound .. bound,
    those beyond going with the outermost (``log_buckets``); without it every offset has its own, num = 2 bound + 1, which is
    the bias of ``RPE``.  Without a table there is no bias.  Finite entries beyond 2.9e37 in size count as that: a row whose every key is masked
    by a type's lowest value attends to its least masked keys, one whose every key is masked by minus infinity is NaN.

    status: a device status word of the caller's (``ops.new_status``), in which a plan, coordinates or buckets out of range are reported; the caller
    checks it when the host next waits.  Without one the call checks for itself and waits for the device.
    Gradients: qkv and table."""
    _same_device(qkv, order_row, pad, unpad, cu_seqlens, grid_coord, table, buckets, status)
    _check_qkv(qkv, heads)
    bias = None
    if table is not None:
        if grid_coord is None:
            raise ValueError("a bias needs grid_coord")
        if table.dim() != 2 or table.shape[1] != heads or table.shape[0] % 3 or not table.shape[0]:
            raise ValueError("table must be (3 buckets, %d heads), got %s" % (heads, tuple(table.shape)))
        _lib.dtype_id(table)
        num = table.shape[0] // 3
        entries = num if buckets is None else buckets.numel()
        if entries % 2 == 0 or entries > 2 * BUCKETS_MAX_BOUND + 1 or num > entries:
            raise ValueError("%d buckets of %d offsets: an odd number of offsets up to %d, and no more buckets" % (
                num, entries, 2 * BUCKETS_MAX_BOUND + 1))
        if buckets is not None:
            buckets = _int32(buckets, (entries,), "buckets")
        bias = (_int32(grid_coord, (qkv.shape[0], 3), "grid_coord"), buckets, entries // 2, num)
    elif grid_coord is not None or buckets is not None:
        raise ValueError("a bias needs a table")
    return _attend(qkv, table, order_row, pad, unpad, cu_seqlens, bias, heads, max_seqlen, scale, 1, status)


def attention_diff(qkv, lam, order_row, pad, unpad, cu_seqlens, heads, max_seqlen, scale=None, status=None):
    """Differential attention within patches: (N, C) = (softmax(scale q1 k1^T) - lam softmax(scale q2 k2^T)) v.

    qkv (N, 3C), split (3, heads, D), D in 16, 32, 64, bf16 or fp32, where the D values of a head's query are q1 and q2 of
    D / 2 each, its key's k1 and k2; lam (heads,), fp32 or bf16; scale: (D / 2) ** -0.5.  The other arguments as for
    ``attention_bias``.  Gradients: qkv and lam."""
    _same_device(qkv, lam, order_row, pad, unpad, cu_seqlens, status)
    _check_qkv(qkv, heads)
    if lam.shape != (heads,):
        raise ValueError("lam must be (%d,), got %s" % (heads, tuple(lam.shape)))
    _lib.dtype_id(lam)
    return _attend(qkv, lam, order_row, pad, unpad, cu_seqlens, None, heads, max_seqlen, scale, 2, status)
