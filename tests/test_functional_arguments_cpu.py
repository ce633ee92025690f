"""What the trainable operators ask of their arguments: what is refused on the host, and what kernels may not assume."""
import ctypes
import os
import re
import subprocess

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from conftest import ROOT
from pointtransformerv3_b200 import _lib
from pointtransformerv3_b200 import functional as F


def _source(name):
    text = open(os.path.join(ROOT, "pointtransformerv3_b200", "csrc", name)).read()
    return re.sub(r"//[^\n]*", "", text)


def test_norm_weights_are_read_value_by_value():
    """A contiguous slice of a bf16 buffer may start on any 2 bytes: a wider load of it would be a misaligned one."""
    wide = re.findall(r"\(const (?:uint32_t|uint64_t|float2|float4|uint2|uint4|__nv_bfloat162)\s*\*\)\s*(\w[\w.]*)",
                      _source("qk_norm_rope.cu"))
    assert not {"weights", "a.qw", "a.kw"} & set(wide), wide


@pytest.mark.parametrize("dtype,step", [(_lib.DTYPE_IDS[t], t.itemsize) for t in _lib.DTYPE_IDS])
def test_weights_off_their_own_type_are_refused(dtype, step):
    """Before anything is launched: a made-up address between two values."""
    lib = _lib.load()
    rows = 1 << 20
    for q, k in ((rows + step // 2, rows), (rows, rows + step // 2)):
        for call in (lambda: lib.ptv3_qk_norm_rope_fwd(rows, q, k, dtype, None, rows, 1, 16, 1, 1e-6, 100.0, dtype, None),
                     lambda: lib.ptv3_qk_norm_rope_bwd(rows, q, k, dtype, None, rows, rows, rows, rows, 1, 16, 1, 1e-6, 100.0,
                                                       dtype, rows, 1 << 20, None)):
            with pytest.raises(_lib.Ptv3Error, match="unaligned weights"):
                _lib.check(call(), "ptv3_qk_norm_rope")


@pytest.fixture(scope="module")
def place_lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("hostmath") / "libpatch_place_host.so")
    subprocess.check_call(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", "-o", so,
                           os.path.join(ROOT, "tests", "hostmath", "patch_place_host.cpp")])
    return ctypes.CDLL(so)


@pytest.fixture(scope="module")
def places(place_lib):
    lib = place_lib
    i, p = ctypes.c_int, ctypes.c_void_p
    lib.host_places.argtypes = [p, p, ctypes.c_int64, i, i, i, i, i, i, p]

    def call(mine, other, lowest, extent, first, reach, sign, step):
        out = np.empty(mine.size, dtype=np.int32)
        lib.host_places(mine.ctypes.data, other.ctypes.data, mine.size, lowest, extent, first, reach, sign, step, out.ctypes.data)
        return out
    return call


@pytest.mark.parametrize("lowest,extent", [(0, 0), (0, 11), (-40, 117), (2 ** 22, 0), (-2 ** 22, 2 ** 23)])
def test_look_ups_stay_in_the_table_whatever_the_coordinates_are(places, lowest, extent):
    """The plan's rows hold a sequence's box.  Points of the box find the entry of their offset; coordinates that have changed since,
    anything of 32 bits, find some entry of the table.  (Of the largest extent only what is held within the table afterwards
    is computed: no sum passes 32 bits.)"""
    rng = np.random.default_rng(7)
    step, first = 5 + 2, 51200 + 4 * 31
    inside = rng.integers(lowest, lowest + extent + 1, size=(2, 5000)).astype(np.int32)
    ends = np.array([-2 ** 31, 2 ** 31 - 1, 0, lowest, lowest + extent], dtype=np.int32)
    outside = rng.integers(-2 ** 31, 2 ** 31, size=(2, 5000)).astype(np.int32)
    outside[0, :25], outside[1, :25] = np.repeat(ends, 5), np.tile(ends, 5)
    reach = min(extent, 1024)
    for sign in (1, -1):
        got = places(inside[0], inside[1], lowest, extent, first, reach, sign, step)
        want = first + ((reach + sign * (inside[0].astype(np.int64) - inside[1])) << step)
        assert (got == want).all()
        got = places(outside[0], outside[1], lowest, extent, first, reach, sign, step)
        far = (extent - reach) << step              # (beyond the table only where look-ups are held afterwards)
        assert got.min() >= first - far and got.max() <= first + ((2 * reach) << step) + far


@pytest.mark.parametrize("rows", [64, 128, 256])
def test_blocks_of_keys_have_numbers_of_their_own(place_lib, rows):
    """Numbered by rows, all blocks that leave a share of a table's gradient, and the numbers that are cleared, are each number below
    n_pad / rows + n_seq once: the sum behind them reads nothing that was not written."""
    rng = np.random.default_rng(rows)
    out = np.empty(4096, dtype=np.int64)
    for lengths in ([0], [1], [rows], [rows - 1, 1], [0, 0, 5 * rows + 3, 0], [20] * 500 + [1024], list(rng.integers(0, 700, 300)),
                    list(rng.integers(0, 3, 300)), [rows * 7] * 20):
        start, got = 0, []
        for seq, n in enumerate(lengths):
            count = place_lib.host_bins(start, int(n), rows, seq, ctypes.c_void_p(out.ctypes.data))
            got += out[:count].tolist()
            start += int(n)
        assert got == list(range(start // rows + len(lengths)))


def _workspace(n, n_pad, n_seq, longest, heads, bound, dtype):
    args = _lib.PATCH_ATTENTION_ARGS.pack(n, n_pad, n_seq, longest, 16 * heads, heads, 1, dtype, 0.25, bound, 2 * bound + 1, 0, 0,
                                          *([1 << 20] * 5), 1 << 20, 0, 1 << 20, 0, *([1 << 20] * 4), 0, 1 << 20, 1 << 20,
                                          1 << 20, 0, 0, 0)
    return _lib.load().ptv3_patch_attention_workspace_bytes(args)


@pytest.mark.parametrize("dtype", [0, 1])
def test_workspace_follows_the_rows(dtype):
    """Many short sequences beside a long one: the table's gradient takes space for the blocks that there are, a number for each
    sequence and one for every 64 rows at most; and of whole patches alone no more than their blocks."""
    n, seqs, heads, bound = 400000 + 1500, 20002, 4, 512
    entries = heads * 3 * (2 * bound + 1) * 4
    per_row = 4 * (2 * heads + heads * 16 * 4)
    got = _workspace(n, n + 548, seqs, 1024, heads, bound, dtype)
    assert 0 < got <= (seqs + (n + 548) / 64) * entries * 65 / 64 + (n + 548) * per_row
    got = _workspace(100 * 1024, 100 * 1024, 100, 1024, heads, bound, dtype)
    assert 0 < got <= 100 * 1024 / 64 * entries * 65 / 64 + 100 * 1024 * per_row


class _Cuda(torch.Tensor):
    """A CPU tensor that says it is on the GPU, for checks that come before any kernel."""
    is_cuda = True


def t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_Cuda)


def plan(n=8):
    return [t(n, dtype=torch.int64) for _ in range(3)] + [t(2, dtype=torch.int32)]


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("call", [
    lambda d: F.qk_norm_rope(d(t(8, 48)), 1, None, t(16), t(16)),
    lambda d: F.qk_norm_rope(t(8, 48), 1, None, d(t(16)), t(16)),
    lambda d: F.qk_norm_rope(t(8, 48), 1, None, t(16), d(t(16))),
    lambda d: F.attention_bias(d(t(8, 48)), *plan(), 1, 8),
    lambda d: F.attention_bias(t(8, 48), *plan(), 1, 8, grid_coord=t(8, 3, dtype=torch.int32), table=d(t(9, 1))),
    lambda d: F.attention_diff(d(t(8, 48)), t(1), *plan(), 1, 8),
    lambda d: F.attention_diff(t(8, 48), d(t(1)), *plan(), 1, 8),
])
def test_tangents_are_refused(call, grad):
    """Forward-mode derivatives would be lost, with a graph and without one."""
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(lambda x: forward_ad.make_dual(x.requires_grad_(grad), torch.ones_like(x)))


def test_a_level_without_tangents_is_no_reason_to_refuse():
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="max_seqlen"):          # (the check behind)
            F.attention_bias(t(8, 48), *plan(), 1, 0)
