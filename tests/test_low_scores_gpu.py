"""Rows whose every score is far below zero, down to the lowest values of a type: softmax of what is least masked, with its
gradients (bounds on norms: functional_norms.py)."""
import pytest
import torch

import functional_norms as N
import functional_reference as R
from pointtransformerv3_b200 import functional as F
from test_functional_gpu import DTYPES, IDS, geometry, normal, plan

pytestmark = pytest.mark.gpu


def hold(p, width, H, dtype, table, bound):
    C = width * H
    qkv, dout = normal(p["n"], 3 * C, seed=1, dtype=dtype), normal(p["n"], C, seed=3, dtype=dtype)
    x, w = qkv.clone().requires_grad_(), table.clone().requires_grad_()
    out = F.attention_bias(x, *geometry(p), H, p["longest"], grid_coord=p["grid"], table=w)
    got = (out,) + torch.autograd.grad(out, (x, w), dout)
    ref = R.attention(qkv, *geometry(p), H, width ** -0.5, 1, table, p["grid"], bound, None, dout)
    for name, t in zip(("out", "dqkv", "dparam"), got):
        N.check(t.detach(), ref, name, qkv, dout, dtype)
    with torch.no_grad():
        assert torch.equal(out, F.attention_bias(qkv, *geometry(p), H, p["longest"], grid_coord=p["grid"], table=table))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("width,H", [(16, 2), (32, 1), (64, 1)])
@pytest.mark.parametrize("low", [float(torch.finfo(torch.bfloat16).min), -1e37, -1e31, float(torch.finfo(torch.bfloat16).max)])
def test_tables_of_one_value(low, width, H, dtype):
    """All keys alike: a score that small (or that large) has no bits for q.k, in 64 bits neither, and a row is the mean of its values."""
    p = plan([300, 41], 128)
    hold(p, width, H, dtype, torch.full((3 * 15, H), low, device="cuda"), 7)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("width,H", [(16, 2), (32, 1), (64, 1)])
@pytest.mark.parametrize("table_dtype", [torch.float32, torch.bfloat16], ids=["table32", "table16"])
def test_masks_that_leave_some_rows_without_a_key(table_dtype, width, H, dtype):
    """Entries of the type's lowest value at about half of the offsets, that of zero among them: rows with keys of no, one, two and
    three such entries.  Some more entries are minus infinity, which nothing makes up for."""
    p = plan([260, 300], 128, extent=9)
    g = torch.Generator().manual_seed(5)
    table = normal(3 * 11, H, seed=2, scale=0.5)
    lowest = torch.rand(33, H, generator=g).cuda() < 0.5
    lowest[[5, 16]] = True
    table = torch.where(lowest, torch.finfo(table_dtype).min, table)
    table[[0, 12, 30]] = float("-inf")
    hold(p, width, H, dtype, table.to(table_dtype), 5)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_products_below_the_range_of_masks(dtype):
    """Scores of -2^102 without a bias, the same for all keys: the mean of the values, and their gradient."""
    p = plan([200, 33], 64)
    width, n = 16, p["n"]
    qkv, dout = normal(n, 48, seed=1, dtype=dtype), normal(n, width, seed=2, dtype=dtype)
    qkv[:, :16], qkv[:, 16:32] = 2.0 ** 50, -2.0 ** 50
    x = qkv.clone().requires_grad_()
    out = F.attention_bias(x, *geometry(p), 1, p["longest"])
    ref = R.attention(qkv, *geometry(p), 1, 0.25, dout=dout)
    values = torch.ones(1, device="cuda")               # (the floor goes by the features' size, here that of values: about 4)
    N.check(out.detach(), ref, "out", 4 * values, dout, dtype)
    dv = torch.autograd.grad(out, x, dout)[0][:, 32:]
    N.check(dv, {"dv": (ref["dqkv"][0][:, 32:],)}, "dv", 4 * values, dout, dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("level", [300.0, -5000.0, 70000.0])
def test_gradients_at_a_level(level, dtype):
    """One entry's value added to every score changes nothing but its rounding: 2^-24 of the level for each score, which all
    probabilities of a row share as their relative error, forward and backward alike."""
    p = plan([700, 41], 512)
    H, C = 2, 32
    qkv, dout = normal(p["n"], 3 * C, seed=1, dtype=dtype), normal(p["n"], C, seed=3, dtype=dtype)
    table = normal(3 * 15, H, seed=2, scale=0.5)
    table[:15] = level
    x, w = qkv.clone().requires_grad_(), table.clone().requires_grad_()
    out = F.attention_bias(x, *geometry(p), H, p["longest"], grid_coord=p["grid"], table=w)
    got = (out,) + torch.autograd.grad(out, (x, w), dout)
    ref = R.attention(qkv, *geometry(p), H, 0.25, 1, table, p["grid"], 7, None, dout)
    for name, t in zip(("out", "dqkv", "dparam"), got):
        for part, err, bound in N.errors(t.detach(), ref, name, qkv, dout, dtype):
            value = dict(N.parts(name, ref[name][0]))[part]
            # two roundings of a score in powers of two (1.45 times the level), half a step each, and log 2 back: 2 2^-24 of it
            assert err <= bound + 2 * 2.0 ** -24 * abs(level) * float(value.norm()), (part, err, bound)
