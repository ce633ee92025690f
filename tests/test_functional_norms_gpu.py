"""Norms of what results and gradients of patch attention are off by (functional_norms.py), where the elementwise bounds are wide: patches
of several windows of a table's gradient, of 512 and 1 024 rows, and launches whose warps own two row tiles."""
import pytest
import torch

import functional_norms as N
from pointtransformerv3_b200 import functional as F
from test_functional_gpu import DTYPES, IDS, PLANS, geometry, normal, plan, run_bias, run_diff
import functional_reference as R

pytestmark = pytest.mark.gpu


def hold(p, got, ref, qkv, dout, dtype, what):
    for name, t in zip(("out", "dqkv", "dparam"), got):
        N.check(t.detach(), ref, name, qkv, dout, dtype, what)


def inputs(p, C, dtype, seed):
    """qkv and the result's gradient as run_bias and run_diff make them."""
    return normal(p["n"], 3 * C, seed=seed).to(dtype), lambda s: normal(p["n"], C, seed=s, dtype=dtype)


def both(p, width, H, dtype, bound=7, **kw):
    C = width * H
    qkv, dout = inputs(p, C, dtype, 1)
    *got, ref = run_bias(p, C, H, dtype, dtype, bound, **kw)
    hold(p, got, ref, qkv, dout(3), dtype, "bias, width %d" % width)
    qkv, dout = inputs(p, C, dtype, 5)
    *got, ref = run_diff(p, C, H, dtype, torch.float32)
    hold(p, got, ref, qkv, dout(6), dtype, "two maps, width %d" % width)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("counts,patch", PLANS + [([1400, 800], 512), ([2048, 5], 1024)], ids=lambda v: str(v)[:20])
def test_norms(counts, patch, dtype):
    p = plan(counts, patch)
    for width, H in ((16, 3), (32, 1), (64, 2)):
        both(p, width, H, dtype)
    C = 32
    qkv = normal(p["n"], 3 * C, seed=3, dtype=dtype).requires_grad_()
    dout = normal(p["n"], C, seed=4, dtype=dtype)
    out = F.attention_bias(qkv, *geometry(p), 2, p["longest"])
    got = (out,) + torch.autograd.grad(out, qkv, dout)
    hold(p, got, R.attention(qkv.detach(), *geometry(p), 2, 0.25, dout=dout), qkv.detach(), dout, dtype, "plain")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("width,H", [(16, 17), (32, 9), (64, 8), (64, 11)])
def test_norms_of_long_launches(width, H, dtype):
    both(plan([3000, 1100], 512), width, H, dtype, 9)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("log", [False, True])
def test_norms_of_a_table_with_far_entries(log, dtype):
    p = plan([1100], 1024, extent=300)
    buckets, num = F.log_buckets(200, device="cuda") if log else (None, None)
    qkv, dout = inputs(p, 32, dtype, 1)
    *got, ref = run_bias(p, 32, 2, dtype, dtype, 200, buckets, num)
    hold(p, got, ref, qkv, dout(3), dtype, "far")
