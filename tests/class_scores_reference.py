"""Scores of logits and losses against a teacher's lists in 64 bits, and how far 32-bit results may be from them.

Every function takes logits as they are given to the operators, on any device, and returns doubles.  A tolerance counts the roundings
of the formula as the operators' documentation states it: U = 2^-24 for each of fp32, 4 U for the exponential unit and 2^-21 for a logarithm on
it, n U for a sum of n values one after another (64 at most on a thread, or a 256th of the row, then the threads'), and half a step of the
output's type."""
import math

import torch

U = 2.0 ** -24
INF = math.inf


def _sum_error(K):
    return (max(64, -(-K // 256)) + 16) * U


def log_softmax(x, temperature):
    """(log p, log S) of rows of doubles; a row of masked classes alone: minus infinity."""
    m = x.amax(1, keepdim=True)
    z = (x - torch.where(m == -INF, 0.0, m)) / temperature
    log_s = torch.log(torch.exp(z).sum(1, keepdim=True))
    return torch.where(log_s == -INF, -INF, z - log_s), log_s


def _p_error(p, logp, log_s, K):
    """Of a probability, as a share of it."""
    return _sum_error(K) + 8 * U * (2 + torch.where(p > 0, -logp, 0.0) + log_s.clamp_min(0))


def scores(logits, labels=None, top=0, temperature=1.0, ignore_index=-1, upstream=None):
    """dict name -> (value, tolerance) of log_prob, entropy, top_log_probs, top_classes (no tolerance) and, with upstream = the gradients of
    the first three or None each, dlogits."""
    x = logits.double()
    n, K = x.shape
    logp, log_s = log_softmax(x, temperature)
    p = torch.exp(logp)
    none = log_s[:, 0] == -INF
    plogp = torch.where(p == 0, 0.0, p * logp)
    entropy = -plogp.sum(1)

    def lp_tol(v):
        return _sum_error(K) + 6 * U * torch.where(v == -INF, 0.0, v).abs()
    h_tol = _sum_error(K) * (1 + 4 * entropy) + 4 * U * (1 + entropy) ** 2 + 4 * U * (p * torch.where(p > 0, logp, 0.0) ** 2).sum(1)
    out = dict(entropy=(entropy, h_tol))
    onehot = torch.zeros_like(x)
    if labels is not None:
        there = labels != ignore_index
        valid = there & (labels >= 0) & (labels < K)
        at = torch.where(valid, labels, 0)[:, None].long()
        value = torch.where(there, torch.where(valid, logp.gather(1, at)[:, 0], math.nan), 0.0)
        out["log_prob"] = value, lp_tol(value)
        onehot.scatter_(1, at, valid.double()[:, None])
    k = min(top, K)
    if top:
        order = torch.sort(torch.where(x.isnan(), INF, x + 0.0), dim=1, descending=True, stable=True)[1]
        nan = x.isnan()
        if nan.any():                      # above plus infinity
            rank = torch.where(nan, 2.0, torch.where(x == INF, 1.0, 0.0))
            order = torch.gather(order, 1, torch.sort(rank.gather(1, order), dim=1, descending=True, stable=True)[1])
        order = order[:, :k]
        values = torch.full((n, top), -INF, dtype=torch.float64, device=x.device)
        values[:, :k] = logp.gather(1, order)
        classes = torch.full((n, top), -1, dtype=torch.int32, device=x.device)
        classes[:, :k] = order.int()
        out["top_log_probs"] = values, lp_tol(values)
        out["top_classes"] = classes, None
    if upstream is not None:
        g, h, t = upstream
        zero = torch.zeros(n, dtype=torch.float64, device=x.device)
        g = zero if g is None else g.double() * onehot.sum(1)
        h = zero if h is None else h.double()
        direct = onehot * g[:, None]
        size, total = direct.abs(), g.clone()
        a_size = g.abs()
        if t is not None:
            direct = direct.scatter_add(1, order, t.double()[:, :k])
            size = size.scatter_add(1, order, t.double()[:, :k].abs())
            total = total + t.double()[:, :k].sum(1)
            a_size = a_size + t.double()[:, :k].abs().sum(1)
        a = -total - h * entropy
        dx = (p * a[:, None] - h[:, None] * plogp + direct) / temperature
        a_tol = (top + 4) * U * (a_size + (h * entropy).abs()) + h.abs() * h_tol
        lp = torch.where(p > 0, logp, 0.0)
        dense = p * (a.abs()[:, None] + h.abs()[:, None] * lp.abs())
        tol = dense * (_p_error(p, lp, log_s, K) + 8 * U) + p * (a_tol[:, None] + h.abs()[:, None] * (_sum_error(K) + 8 * U * (1 + lp.abs())))
        tol = (tol + 8 * U * size) / temperature
        dx = torch.where(none[:, None], 0.0, dx)
        # numbers below 2^-126 are zero on the way: p and its products, of which p a and p h log p (|log p| up to 110) are two
        flushed = 2.0 ** -126 * (4 + a.abs() + 110 * h.abs())[:, None] / temperature
        tol = torch.where(none[:, None], 0.0, tol + flushed) + torch.finfo(logits.dtype).eps / 2 * dx.abs() * (1 + 1e-3) + 1e-37
        out["dlogits"] = dx, tol
    return out


def distill(logits, teacher, classes, temperature=1.0, rest=False, upstream=None):
    """dict name -> (value, tolerance) of loss and, with upstream = its gradient, dlogits."""
    x, v, c = logits.double(), teacher.double(), classes.long()
    n, K = x.shape
    k = c.shape[1]
    logp, log_s = log_softmax(x, temperature)
    none = log_s[:, 0] == -INF
    bad = ((c < -1) | (c >= K)).any(1)
    there = (c >= 0) & (c < K)
    at = torch.where(there, c, 0)
    v = torch.where(there, v, -INF)
    some = there.any(1)
    if rest:
        log_t = v
    else:
        m = v.amax(1, keepdim=True)
        z = (v - torch.where(m == -INF, 0.0, m)) / temperature
        s = torch.exp(z).sum(1, keepdim=True)
        log_t = torch.where(s == 0, -INF, z - torch.log(s))
    t = torch.exp(log_t)
    lt = torch.where(t == 0, 0.0, log_t)
    lp = logp.gather(1, at)
    part = torch.where(t == 0, 0.0, t * (lt - lp))
    loss = part.sum(1)
    t_tol = t * ((k + 12) * U + 4 * U * lt.abs())
    lp_fin = torch.where(lp == -INF, 0.0, lp)
    tol = (t * ((_sum_error(K) + 2.0 ** -20) + 8 * U * (lp_fin.abs() + lt.abs())) + t_tol * (lt - lp_fin).abs()).sum(1)
    tol = tol + (k + 4) * U * torch.where(part.abs() < INF, part.abs(), 0.0).sum(1)
    mass, mass_tol = t.sum(1), t_tol.sum(1) + k * U * t.sum(1)
    inside = torch.zeros(n, K + 1, dtype=torch.bool, device=x.device)
    inside.scatter_(1, torch.where(there, at, K), True)
    inside = inside[:, :-1]
    log_r = t_r = None
    if rest:
        outside = x.masked_fill(inside, -INF)
        open_ = (outside.amax(1) != -INF) & some
        t_r = torch.where(open_, (1 - t.sum(1)).clamp_min(0), 0.0)
        logq, _ = log_softmax(outside, temperature)          # log p_j / p_r
        shift = logp - logq
        log_r = torch.where(outside == -INF, -INF, shift).amax(1)
        others = t.sum(1) - t.amax(1)
        tr_tol = torch.where(open_, (k + 4) * U * others + t_tol.sum(1) - t_tol.gather(1, t.argmax(1, keepdim=True))[:, 0] +
                             4 * U * (t_r + others) + 2 * U, 0.0)
        # (the largest entry's part comes from expm1: right to a few U of 1 - t)
        lr = torch.where(open_, log_r, 0.0)
        ltr = torch.where(t_r > 0, torch.log(t_r.clamp_min(1e-300)), 0.0)
        loss = loss + torch.where(t_r > 0, t_r * (ltr - lr), 0.0)
        low = torch.log(tr_tol.clamp_min(1e-300)).abs()
        tol = tol + t_r * (2 * _sum_error(K) + 2.0 ** -19 + 8 * U * (lr.abs() + ltr.abs()))
        tol = tol + tr_tol * (1 + torch.maximum(ltr.abs(), torch.where(tr_tol > 0, low, 0.0)) + lr.abs())
        mass, mass_tol = mass + t_r, mass_tol + tr_tol
    out = dict(loss=(torch.where(bad, math.nan, loss), tol))
    if upstream is not None:
        g = upstream.double()[:, None] / temperature
        p = torch.exp(logp)
        p = torch.where(none[:, None], 0.0, p)
        lpf = torch.where(p > 0, logp, 0.0)
        dx = mass[:, None] * p
        gtol = p * (mass[:, None] * (_p_error(p, lpf, log_s, K) + 4 * U) + mass_tol[:, None])
        taken = torch.zeros(n, K + 1, dtype=torch.float64, device=x.device)
        spot = torch.where(there, at, K)
        dx = dx - taken.scatter_add(1, spot, t)[:, :-1]
        gtol = gtol + taken.scatter_add(1, spot, t_tol + (k + 4) * U * t)[:, :-1]
        if rest:
            q = torch.where(inside | ~open_[:, None] | (outside == -INF), 0.0, torch.exp(logq))
            lq = torch.where(q > 0, logq, 0.0)
            dx = dx - q * t_r[:, None]
            f = torch.exp(torch.where(open_, log_r, -INF))
            f_tol = mass * f * (2 * _sum_error(K) + 2.0 ** -20 + 8 * U * (lr.abs() + log_s[:, 0].clamp_min(0)))
            gtol = gtol + q * (tr_tol + f_tol + mass_tol * f)[:, None]
            share = _sum_error(K) + 2.0 ** -20 + 8 * U * (2 + lq.abs() + lr.abs()[:, None] + log_s.clamp_min(0))
            gtol = gtol + (mass * f + t_r)[:, None] * q * share
        dx = torch.where(none[:, None], 0.0, dx * g)
        gtol = gtol * g.abs() * 1.01 + 4 * U * dx.abs()
        out["dlogits"] = dx, gtol + torch.finfo(logits.dtype).eps / 2 * dx.abs() * (1 + 1e-3) + 1e-37
    return out


def assert_near(got, want, tol, what=""):
    """Within the tolerance, equal where it is infinite, NaN where it is.  What is beyond the largest number of fp32 is infinite there."""
    got, want = got.double().cpu(), want.double().cpu()
    want = torch.where(want.abs() > torch.finfo(torch.float32).max, torch.copysign(torch.tensor(INF).double(), want), want)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(got.isnan(), want.isnan()), what
    there = ~want.isnan()
    assert torch.equal(got.isinf() & there, want.isinf() & there) and torch.equal(got[got.isinf()], want[want.isinf()]), what
    there &= ~want.isinf()
    off = (got - want).abs()[there] - tol.double().cpu()[there]
    if off.numel() and off.max() > 0:
        worst = int(off.argmax())
        raise AssertionError("%s: %g for %g, beyond %g" % (what, got[there][worst], want[there][worst], tol.double().cpu()[there][worst]))
