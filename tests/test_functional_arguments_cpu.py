"""What the trainable operators ask of their arguments: what is refused on the host, and what kernels may not assume."""
import os
import re

import pytest

from conftest import ROOT
from pointtransformerv3_b200 import _lib


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
