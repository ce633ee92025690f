"""The bounds on norms reject gradients that are wrong as a whole, at every plan that the GPU tests use."""
import itertools

import pytest
import torch

import functional_norms as N
import functional_reference as R


def plan(counts, patch, seed=0, extent=12):
    """Random order, whole patches whose last one borrows rows of the one before, scenes shorter than a patch as they are."""
    g = torch.Generator().manual_seed(seed)
    order, pad, unpad, cu, at, end = [], [], [], [0], 0, 0
    for c in counts:
        order.append(torch.randperm(c, generator=g) + at)
        whole = -(-c // patch) * patch if c > patch else c
        p = torch.arange(at, at + whole)
        if whole > c:
            p[c:] = p[c - patch:whole - patch].clone()
        pad.append(p)
        unpad.append(torch.arange(end, end + c))
        cu += list(range(end + patch, end + whole, patch)) + [end + whole]
        at, end = at + c, end + whole
    grid = torch.randint(0, extent, (at, 3), generator=g, dtype=torch.int32)
    return at, (torch.cat(order), torch.cat(pad), torch.cat(unpad), torch.tensor(cu, dtype=torch.int32)), grid


PLANS = [([1], 16), ([65], 64), ([1, 127, 3], 64), ([17] * 9, 48), ([333, 200], 111), ([1024], 1024), ([1500], 1024),
         ([70, 1, 900], 257), ([1400, 800], 512)]


@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("counts,patch", PLANS, ids=lambda v: str(v)[:20])
def test_wrong_gradients_are_rejected(counts, patch, maps):
    n, geometry, grid = plan(counts, patch)
    H, W = 2, 16
    g = torch.Generator().manual_seed(1)
    qkv, dout = torch.randn(n, 3 * H * W, generator=g), torch.randn(n, H * W, generator=g)
    param = 0.5 * torch.randn(*((3 * 15, H) if maps == 1 else (H,)), generator=g)
    ref = R.attention(qkv, *geometry, H, (W // maps) ** -0.5, maps, param, grid, 7, None, dout)
    for name, dtype in itertools.product(("out", "dqkv", "dparam"), (torch.float32, torch.bfloat16)):
        right = ref[name][0]
        N.check(right, ref, name, qkv, dout, dtype)
        N.check(right.to(dtype), ref, name, qkv, dout, dtype)            # (stored in its type)
        for wrong in (torch.zeros_like(right), -right, 0.9 * right, 0.97 * right):
            for part, err, bound in N.errors(wrong, ref, name, qkv, dout, dtype):
                degenerate = n == 1 and (part in ("dq", "dk") or (part == "dparam" and maps == 1))
                assert err > bound or degenerate, (part, err, bound)
