"""What the trainable operators refuse before anything is launched, and their host arithmetic."""
import itertools

import pytest
import torch

import functional_reference as R
from pointtransformerv3_b200 import _lib
from pointtransformerv3_b200 import functional as F


class _Cuda(torch.Tensor):
    """A CPU tensor that says it is on the GPU, for checks that come before any kernel."""
    is_cuda = True


def t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_Cuda)


def args(n=8, n_pad=8):
    i = torch.int64
    return [t(n, dtype=i), t(n_pad, dtype=i), t(n, dtype=i), t(2, dtype=torch.int32)]


def test_cpu_tensors_are_refused():
    with pytest.raises(_lib.Ptv3Error, match="no CPU path"):
        F.qk_norm_rope(torch.zeros(4, 48), 1, torch.zeros(4, 3))
    with pytest.raises(_lib.Ptv3Error, match="no CPU path"):
        F.attention_bias(torch.zeros(8, 48), *[x.as_subclass(torch.Tensor) for x in args()], 1, 8)


@pytest.mark.parametrize("call,word", [
    (lambda: F.qk_norm_rope(t(4, 47), 1, t(4, 3)), r"\(N, 3C\)"),
    (lambda: F.qk_norm_rope(t(4, 48), 3, t(4, 3)), "3 heads"),
    (lambda: F.qk_norm_rope(t(4, 48), 0, t(4, 3)), "0 heads"),
    (lambda: F.qk_norm_rope(t(4, 48), 1), "or all three"),
    (lambda: F.qk_norm_rope(t(4, 48), 1, None, t(16)), "or all three"),
    (lambda: F.qk_norm_rope(t(4, 48), 1, None, t(16), t(8)), r"\(16,\)"),
    (lambda: F.qk_norm_rope(t(4, 48), 1, None, t(16), t(16, dtype=torch.bfloat16)), "of one type"),
    (lambda: F.qk_norm_rope(t(4, 48), 1, t(3, 3, dtype=torch.int32)), "grid_coord"),
    (lambda: F.qk_norm_rope(t(4, 48), 1, t(4, 3)), "integers"),
    (lambda: F.attention_bias(t(8, 48), *args(), 1, 8, status=t(1)), "int32 word"),
    (lambda: F.attention_bias(t(8, 48), *args(), 1, 8, table=t(9, 1)), "needs grid_coord"),
    (lambda: F.attention_bias(t(8, 48), *args(), 1, 8, grid_coord=t(8, 3)), "needs a table"),
    (lambda: F.attention_bias(t(8, 48), *args(), 1, 8, grid_coord=t(8, 3), table=t(9, 2)), "1 heads"),
    (lambda: F.attention_bias(t(8, 48), *args(), 1, 8, grid_coord=t(8, 3), table=t(8, 1)), "3 buckets"),
    (lambda: F.attention_bias(t(8, 48), *args(), 1, 8, grid_coord=t(8, 3), table=t(6, 1)), "odd number"),
    (lambda: F.attention_bias(t(8, 48), *args(), 1, 8, grid_coord=t(8, 3), table=t(15, 1), buckets=t(3)), "no more buckets"),
    (lambda: F.attention_bias(t(8, 48), *args(), 1, 8, grid_coord=t(8, 3), table=t(3 * 1027, 1)), "up to 1025"),
    (lambda: F.attention_bias(t(8, 48), *args(), 1, 8, grid_coord=t(7, 3), table=t(9, 1)), "grid_coord"),
    (lambda: F.attention_bias(t(8, 72), *args(), 1, 8), "heads of 24"),
    (lambda: F.attention_bias(t(8, 48), *args(7), 1, 8), "order_row"),
    (lambda: F.attention_bias(t(8, 48), *args(8, 7), 1, 8), "pad 8 to 16"),
    (lambda: F.attention_bias(t(8, 48), *args(8, 17), 1, 8), "pad 8 to 16"),
    (lambda: F.attention_bias(t(8, 48), *args()[:3], t(2), 1, 8), "int32"),
    (lambda: F.attention_bias(t(8, 48), t(8), *args()[1:], 1, 8), "int64"),
    (lambda: F.attention_bias(t(8, 48), *args(), 1, 0), "max_seqlen"),
    (lambda: F.attention_diff(t(8, 48), t(2), *args(), 1, 8), "lam"),
    (lambda: F.attention_bias(t(8, 48), *args(), 1, 8, 0.0), "scale"),
    (lambda: F.attention_diff(t(8, 48), t(1), *args(), 1, 8, float("inf")), "scale"),
])
def test_refusals(call, word):
    with pytest.raises(ValueError, match=word):
        call()


def test_other_types_are_refused():
    for call in (lambda: F.qk_norm_rope(t(4, 48, dtype=torch.float16), 1, t(4, 3)),
                 lambda: F.attention_bias(t(8, 48, dtype=torch.float64), *args(), 1, 8),
                 lambda: F.attention_diff(t(8, 48), t(1, dtype=torch.float16), *args(), 1, 8)):
        with pytest.raises(_lib.Ptv3Error, match="not supported"):
            call()


@pytest.mark.parametrize("bound,exact,per_octave", list(itertools.product((1, 2, 7, 8, 9, 20, 128, 512), (1, 8), (1, 4))))
def test_log_buckets(bound, exact, per_octave):
    lut, num = F.log_buckets(bound, exact, per_octave)
    b = lut.tolist()
    assert len(b) == 2 * bound + 1 and num % 2 == 1
    assert sorted(set(b)) == list(range(num)) and b == sorted(b)                  # none empty, in the order of the offsets
    assert all(b[bound + d] + b[bound - d] == num - 1 for d in range(bound + 1))
    assert all(b[bound + d] == num // 2 + d for d in range(min(bound + 1, exact)))


def test_the_references_gradients_are_those_of_differences():
    """The 64-bit forms that the kernels are held to: their hand-written gradients are the slopes of their results."""
    g = torch.Generator().manual_seed(0)
    n, H, W = 13, 2, 4
    order = torch.randperm(n, generator=g)
    pad = torch.tensor(list(range(8)) + [8, 9, 10, 11, 12, 5, 6, 7])
    unpad, cu = torch.arange(n), torch.tensor([0, 8, 16], dtype=torch.int32)
    grid = torch.randint(0, 9, (n, 3), generator=g)
    qkv, dout = (torch.randn(n, c, generator=g, dtype=torch.float64) for c in (3 * H * W, H * W))
    buckets, num = F.log_buckets(5, 2, 2)
    for maps, param in ((1, torch.randn(3 * num, H, generator=g, dtype=torch.float64)), (2, torch.tensor([0.4, -0.7]).double())):
        def f(x, w, dout=None):
            return R.attention(x, order, pad, unpad, cu, H, 0.5, maps, w, grid, 5, buckets, dout)
        res, h = f(qkv, param, dout), 1e-4
        for name, at in (("dqkv", 0), ("dparam", 1)):
            for _ in range(4):
                step = torch.randn((qkv, param)[at].shape, generator=g, dtype=torch.float64)
                ends = []
                for s in (h, -h):
                    moved = [qkv, param]
                    moved[at] = moved[at] + s * step
                    ends.append(float((f(*moved)["out"][0] * dout).sum()))
                assert abs((ends[0] - ends[1]) / (2 * h) - float((res[name][0] * step).sum())) < 1e-5


def test_points_without_sequences_are_refused():
    for ends in (t(1, dtype=torch.int32), t(0, dtype=torch.int32)):
        with pytest.raises(ValueError, match="one sequence"):
            F.attention_bias(t(8, 48), *args()[:3], ends, 1, 8)
