"""Plain 64-bit forms of the operators in ``pointtransformerv3_b200.functional`` and bounds on what rounding may add to them.

The references are autograd graphs over elementary torch operations, sequence by sequence; the bounds are sums of absolute values
times the relative errors that the arithmetic of a type allows (half a step of bf16 2^-8, of fp32 2^-24)."""
import math

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def qk_norm_rope(qkv, heads, grid=None, wq=None, wk=None, eps=1e-6, base=100.0):
    """qkv float64; angles in 64 bits."""
    n, c = qkv.shape[0], qkv.shape[1] // 3
    D = c // heads
    p = D // 6
    parts = []
    for x, w in ((qkv[:, :c], wq), (qkv[:, c:2 * c], wk)):
        x = x.reshape(n, heads, D)
        if w is not None:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + eps) * w
        if grid is not None:
            cols = [x[..., d] for d in range(D)]
            for i in range(3 * p):
                a = (grid[:, i // p].double() * base ** (-(i % p) / p))[:, None]
                u, v = cols[2 * i], cols[2 * i + 1]
                cols[2 * i], cols[2 * i + 1] = u * a.cos() - v * a.sin(), u * a.sin() + v * a.cos()
            x = torch.stack(cols, -1)
        parts.append(x.reshape(n, c))
    return torch.cat(parts + [qkv[:, 2 * c:]], 1)


def bias_of(table, grid_q, grid_k, bound, buckets=None):
    """(heads, queries, keys) of the table's sums."""
    num = table.shape[0] // 3
    out = 0
    for a in range(3):
        off = (grid_q[:, None, a].long() - grid_k[None, :, a].long()).clamp(-bound, bound) + bound
        out = out + table[a * num + (off if buckets is None else buckets.long()[off])]
    return out.permute(2, 0, 1)


def attention(qkv, order, pad, unpad, cu, heads, scale, maps=1, param=None, grid=None, bound=0, buckets=None, dout=None):
    """The result and, with dout, gradients, each with its bound: dict(out, dqkv, dparam), values (tensor, sums), where the
    sums are those that ``tolerances`` turns into a bound.  Everything in float64 on the device of the inputs."""
    n, c = qkv.shape[0], qkv.shape[1] // 3
    W = c // heads
    D = W // maps
    z = dict(dtype=torch.float64, device=qkv.device)
    out, out_p = torch.zeros(n, c, **z), torch.zeros(n, c, **z)
    dqkv, dqkv_p, dqkv_e = (torch.zeros(n, 3 * c, **z) for _ in range(3))
    dparam = None if param is None else torch.zeros_like(param, dtype=torch.float64)
    dparam_e = None if param is None else torch.zeros_like(dparam)
    top = bias_top = 0.0
    answers = torch.full((pad.shape[0],), -1, dtype=torch.int64, device=qkv.device)
    answers[unpad] = order
    ends = cu.tolist()
    for a, b in zip(ends[:-1], ends[1:]):
        if a == b:
            continue
        pts, own = order[pad[a:b]], answers[a:b]
        keep = own >= 0
        q, k, v = (t.reshape(b - a, heads, W).transpose(0, 1) for t in qkv[pts].double().split(c, 1))
        probs, score = [], 0.0
        for m in range(maps):
            qm, km = q[..., m * D:(m + 1) * D], k[..., m * D:(m + 1) * D]
            s = qm @ km.transpose(1, 2) * scale
            size = qm.abs() @ km.abs().transpose(1, 2) * abs(scale)
            if maps == 1 and param is not None:
                bias = bias_of(param.double(), grid[pts], grid[pts], bound, buckets)
                s = s + bias
                largest = torch.where(param.isfinite(), param, 0).double().abs().max()
                size = size + 3 * largest
                bias_top = max(bias_top, float(largest))
            score = max(score, float(size.max()))
            e = torch.exp(s - s.amax(-1, keepdim=True))
            probs.append(e / e.sum(-1, keepdim=True))
        top = max(top, score)
        lam = param.double()[:, None, None] if maps == 2 else None
        mix = probs[0] if maps == 1 else probs[0] - lam * probs[1]
        size = probs[0] if maps == 1 else probs[0] + lam.abs() * probs[1]
        o, o_p = ((t @ u).transpose(0, 1).reshape(b - a, c) for t, u in ((mix, v), (size, v.abs())))
        out[own[keep]], out_p[own[keep]] = o[keep], o_p[keep]
        if dout is None:
            continue
        do = torch.where(keep[:, None], dout.double()[own.clamp_min(0)], 0.0).reshape(b - a, heads, W).transpose(0, 1)
        G, Ga = do @ v.transpose(1, 2), do.abs() @ v.abs().transpose(1, 2)
        grads = [torch.zeros(heads, b - a, W, **z) for _ in range(9)]
        dq, dk, dv, dq_p, dk_p, dv_p, dq_e, dk_e, dv_e = grads
        dv += mix.transpose(1, 2) @ do
        dv_p += size.transpose(1, 2) @ do.abs()
        for m in range(maps):
            P, at = probs[m], slice(m * D, (m + 1) * D)
            coef = 1.0 if m == 0 else -lam
            delta = (P * G).sum(-1, keepdim=True)
            dS = coef * P * (G - delta)
            # what errors of P and G are relative to (these sums are of absolute values, the scale's too)
            err = (P if m == 0 else lam.abs() * P) * (Ga + (P * Ga).sum(-1, keepdim=True))
            dq[..., at] = dS @ k[..., at] * scale
            dk[..., at] = dS.transpose(1, 2) @ q[..., at] * scale
            dq_p[..., at] = dS.abs() @ k[..., at].abs() * abs(scale)
            dk_p[..., at] = dS.abs().transpose(1, 2) @ q[..., at].abs() * abs(scale)
            dq_e[..., at] = err @ k[..., at].abs() * abs(scale)
            dk_e[..., at] = err.transpose(1, 2) @ q[..., at].abs() * abs(scale)
            if maps == 2 and m == 1:
                dparam -= delta.sum((1, 2))
                dparam_e += (P * Ga).sum((1, 2))
            elif param is not None and maps == 1:
                num = param.shape[0] // 3
                # a bin's sum is kept in units of the largest row's, 2^-25 of it or less: half a unit for each pair
                unit = 2.0 ** -25 * float((P * (Ga + (P * Ga).sum(-1, keepdim=True))).sum(-1).max())
                for axis in range(3):
                    off = (grid[pts][:, None, axis].long() - grid[pts][None, :, axis].long()).clamp(-bound, bound) + bound
                    off = (off if buckets is None else buckets.long()[off]).reshape(-1) + axis * num
                    dparam.index_add_(0, off, dS.reshape(heads, -1).t())
                    dparam_e.index_add_(0, off, err.reshape(heads, -1).t())
                    dparam_e.index_add_(0, off, torch.full_like(err.reshape(heads, -1).t(), unit * 2.0 ** 17))
        flat = lambda *t: torch.cat([x.transpose(0, 1).reshape(b - a, c) for x in t], 1)
        dqkv.index_add_(0, pts, flat(dq, dk, dv))
        dqkv_p.index_add_(0, pts, flat(dq_p, dk_p, dv_p))
        dqkv_e.index_add_(0, pts, flat(dq_e, dk_e, dv_p))
    res = dict(top=top, bias_top=bias_top, out=(out, out_p, out_p))
    if dout is not None:
        res["dqkv"] = (dqkv, dqkv_p, dqkv_e)
        if param is not None:
            res["dparam"] = (dparam, torch.zeros_like(dparam), dparam_e)
    return res


def tolerances(res, name, dtype, width, longest, features=None):
    """Bound of every element of res[name], stored as ``dtype`` and computed from ``features``:
    half a step of the stored value; half a bf16 step of every probability or dS that a bf16 product takes; and what fp32
    arithmetic leaves of a probability: scores of ``top`` at most are off by (width + 8) half steps of fp32, and come in twice, as
    score and in the logarithm of the sum, which adds a half step per key; ex2 2^-22 and as much for the logarithm."""
    value, product, sums = res[name]
    features = features or dtype
    e32 = 2.0 ** -24
    eps = 4 * ((width + 8) * e32 * max(1.0, res["top"]) + longest * e32 + 2.0 ** -21) + 2 * width * e32
    rounding = HALF_STEP[torch.bfloat16] if features == torch.bfloat16 else 0.0
    if rounding:      # a table's entries enter bf16 scores as two bf16 parts, 2^-16 of an entry, three to a score; twice as above
        eps += 2 * 3 * 2.0 ** -16 * res["bias_top"]
    return HALF_STEP[dtype] * value.abs() * (1 + 2.0 ** -7) + rounding * 1.01 * product + eps * sums + 1e-30


def check(got, res, name, width, longest, features=None, what=""):
    value = res[name][0]
    tol = tolerances(res, name, got.dtype, width, longest, features)
    err = (got.double() - value).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), "%s %s: %d of %d outside, worst %g of the bound (error %g, largest value %g)" % (
        what, name, int(bad.sum()), bad.numel(), float((err / tol).max()), float(err.max()), float(value.abs().max()))
