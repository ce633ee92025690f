"""Timed cases of the operators that blocks of serialized attention are built and trained from.

* ``qk``: norms of queries and keys for each head with the rotation by grid coordinates in the same pass
  (``functional.qk_norm_rope``);
* ``bias``: patch attention with a learned relative position bias by buckets (``functional.attention_bias``);
* ``diff``: differential patch attention, the difference of two softmax maps with learned weights
  (``functional.attention_diff``).

Each runs forward alone, as a scoring job does, or forward and backward, as a training step does.  Inputs are made on the GPU from
the seed: surfaces in rooms, points in random order, patches along a z-order curve with the framework's
padding (the last patch of a scene borrows rows from the one before; a scene shorter than a patch is one short
sequence).  Sizes follow the levels of the default backbone.
"""
import math

import torch

own = False

BASE = 100.0          # of the rotation's frequencies
EPS = 1e-6            # of the norms


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # the coarse level of one room, scored: a call whose launch and host work are what counts
        dict(name="qk_1757_256", path="qk", train=False, n=1757, channels=256, heads=16, extent=70, dtype="bf16"),
        # the finest decoder level of a batch of four rooms, scored
        dict(name="qk_407k_64", path="qk", train=False, n=407678, channels=64, heads=4, extent=500, dtype="bf16"),
        # the second level of four rooms in a training step
        dict(name="qk_train_105k_128", path="qk", train=True, n=105505, channels=128, heads=8, extent=250,
             dtype="bf16"),
        # a LiDAR frame in fp32, coordinates up to the depth of the codes, heads of 32
        dict(name="qk_train_64k_64_f32", path="qk", train=True, n=64003, channels=64, heads=2, extent=65535,
             dtype="fp32"),
        # the third level of a room, scored: a few patches, ragged
        dict(name="bias_6k_128", path="bias", train=False, n=6760, scenes=1, patch=1024, channels=128, heads=8,
             bound=31, log=False, dtype="bf16"),
        # the finest level of a room, scored
        dict(name="bias_120k_64", path="bias", train=False, n=120000, scenes=1, patch=1024, channels=64, heads=4,
             bound=31, log=False, dtype="bf16"),
        # the same in a training step, two rooms, far offsets in buckets that widen
        dict(name="bias_train_100k_64", path="bias", train=True, n=100001, scenes=2, patch=1024, channels=64,
             heads=4, bound=128, log=True, dtype="bf16"),
        # fp32 training of a small room
        dict(name="bias_train_12k_32_f32", path="bias", train=True, n=12007, scenes=3, patch=256, channels=32,
             heads=2, bound=20, log=False, dtype="fp32"),
        # a coarse level of one room, scored: one patch and a bit
        dict(name="diff_1560_256", path="diff", train=False, n=1560, scenes=1, patch=1024, channels=256, heads=16,
             dtype="bf16"),
        # the finest level of a room, scored
        dict(name="diff_120k_64", path="diff", train=False, n=120000, scenes=1, patch=1024, channels=64, heads=2,
             dtype="bf16"),
        # a training step of the finest level, two rooms
        dict(name="diff_train_100k_64", path="diff", train=True, n=100001, scenes=2, patch=1024, channels=64, heads=4,
             dtype="bf16"),
        # fp32 training of four short scenes in odd patches
        dict(name="diff_train_20k_64_f32", path="diff", train=True, n=20011, scenes=4, patch=333, channels=64, heads=2,
             dtype="fp32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    path = rng.choice(("qk", "bias", "diff"))
    train, dtype = rng.random() < 0.5, "fp32" if rng.random() < 0.3 else "bf16"
    width = rng.choice((16, 16, 16, 32, 64))
    if path == "qk":
        heads = rng.choice((1, 2, 4, 8, 16))
        n = _log(rng, 200, 26000000 // (width * heads * (4 if train or dtype == "fp32" else 1)))
        return dict(path=path, train=train, n=min(n, 400000), channels=width * heads, heads=heads,
                    extent=_log(rng, 30, 65535), dtype=dtype)
    heads = rng.choice((1, 2, 3, 4, 8))
    patch = rng.choice((1024, 1024, _log(rng, 48, 1024)))
    # rows x keys x channels, as the largest listed case of its kind has at most
    most = 5000000000 if dtype == "bf16" else 400000000
    n = min(100000, _log(rng, 100, most // (patch * width * heads)))
    case = dict(path=path, train=train, n=n, scenes=rng.randint(1, min(8, n // 50)), patch=patch, channels=width * heads,
                heads=heads, dtype=dtype)
    if path == "bias":
        log = rng.random() < 0.5
        case.update(bound=rng.randint(64, 256) if log else rng.randint(4, 64), log=log)
    return case


# --------------------------------------------------------------------------- inputs
def _counts(case):
    """Points of every scene; of three and more the second is a single point."""
    k = case["scenes"]
    weights = [1.0 + 0.6 * (0.618 * (i + 1) % 1.0) for i in range(k)]
    left = case["n"] - (1 if k > 2 else 0)
    if k > 2:
        weights[1] = 0.0
    counts = [int(left * w / sum(weights)) for w in weights]
    if k > 2:
        counts[1] = 1
    counts[0] += case["n"] - sum(counts)
    return counts


def _lengths(case):
    """Sequence lengths: whole patches, or a scene shorter than a patch as it is."""
    out = []
    for c in _counts(case):
        out += [c] if c <= case["patch"] else [case["patch"]] * (-(-c // case["patch"]))
    return out


def _buckets(bound):
    """Buckets of the offsets -bound .. bound: single up to 8, then widening with the logarithm; and their number."""
    d = torch.arange(-bound, bound + 1, dtype=torch.float64)
    far = 8 + torch.floor(torch.log(d.abs().clamp_min(8) / 8) / math.log(2) * 4)
    b = torch.where(d.abs() < 8, d.abs(), far).long()
    half = int(b.max())
    return (b * torch.sign(d).long() + half).int(), 2 * half + 1


def _geometry(case, g):
    """Point order, padding and coordinates of a batch of rooms."""
    counts, patch, dev = _counts(case), case["patch"], "cuda"
    n = sum(counts)
    scene = torch.arange(len(counts), device=dev).repeat_interleave(torch.tensor(counts, device=dev))
    # floors and walls whose cells are about half occupied
    extent = torch.tensor([max(4.0, math.sqrt(c / 2.0)) for c in counts], device=dev)[scene]
    grid = (torch.rand(n, 3, device=dev, generator=g) * extent[:, None]).int()
    axis = torch.randint(0, 3, (n, 1), device=dev, generator=g)
    grid.scatter_(1, axis, (grid.gather(1, axis) // 16) * 16)
    code = scene << 48
    for bit in range(11):
        for a in range(3):
            code = code | (((grid[:, a].long() >> bit) & 1) << (3 * bit + a))
    order = torch.argsort(code, stable=True)
    pad, unpad, cu, at, end = [], [], [0], 0, 0
    for c in counts:
        whole = -(-c // patch) * patch if c > patch else c
        p = torch.arange(at, at + whole)
        if whole > c:
            p[c:] = p[c - patch:whole - patch].clone()
        pad.append(p)
        unpad.append(torch.arange(end, end + c))
        cu += [end + v for v in range(patch, whole, patch)] + [end + whole]
        at, end = at + c, end + whole
    return dict(order=order, pad=torch.cat(pad).to(dev), unpad=torch.cat(unpad).to(dev), grid=grid,
                cu=torch.tensor(cu, dtype=torch.int32, device=dev), longest=max(_lengths(case)))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = torch.float32 if case["dtype"] == "fp32" else torch.bfloat16
    n, c, h = case["n"], case["channels"], case["heads"]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)
    st = dict(case=case, dtype=dtype)
    qkv = normal(n, 3 * c)
    if case["path"] == "qk":
        # rows of different sizes, as a Linear layer gives them
        st["qkv"] = (qkv * (0.3 + 2 * torch.rand(n, 1, device="cuda", generator=g))).to(dtype)
        st["grid"] = torch.randint(0, case["extent"] + 1, (n, 3), device="cuda", generator=g).int()
        st["weights"] = [(1 + 0.2 * normal(c // h)).to(dtype) for _ in range(2)]
        if case["train"]:
            st["dout"] = normal(n, 3 * c).to(dtype)
        return st
    # values of a channel have a mean of their own, as those behind a bias do
    qkv[:, 2 * c:] += 0.5 * normal(c)
    st["qkv"] = qkv.to(dtype)
    st.update(_geometry(case, g))
    st["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    if case["path"] == "bias":
        num = 2 * case["bound"] + 1
        st["buckets"] = None
        if case["log"]:
            lut, num = _buckets(case["bound"])
            st["buckets"] = lut.cuda()
        st["table"] = (0.5 * normal(3 * num, h)).to(dtype)
    else:
        st["lam"] = 0.2 + 0.6 * torch.rand(h, device="cuda", generator=g)
    if case["train"]:
        st["dout"] = normal(n, c).to(dtype)
    return st


# --------------------------------------------------------------------------- one pass
def run(st):
    case = st["case"]
    if own:
        return _run_own(st, case)
    if case["path"] == "qk":
        return _qk_plain(st, case)
    return _attention_plain(st, case)


def _run_own(st, case):
    from pointtransformerv3_b200 import functional as F
    if case["path"] == "qk":
        params = [st["qkv"]] + st["weights"]

        def call(qkv, wq, wk):
            return F.qk_norm_rope(qkv, case["heads"], st["grid"], wq, wk, eps=EPS, base=BASE)
    else:
        geometry = (st["order"], st["pad"], st["unpad"], st["cu"], case["heads"], st["longest"])
        if case["path"] == "bias":
            params = [st["qkv"], st["table"]]

            def call(qkv, table):
                return F.attention_bias(qkv, *geometry, grid_coord=st["grid"], table=table, buckets=st["buckets"],
                                        status=st["status"])
        else:
            params = [st["qkv"], st["lam"]]

            def call(qkv, lam):
                return F.attention_diff(qkv, lam, *geometry, status=st["status"])
    if not case["train"]:
        with torch.no_grad():
            return call(*params)
    leaves = [p.detach().requires_grad_() for p in params]
    out = call(*leaves)
    return (out.detach(),) + torch.autograd.grad(out, leaves, st["dout"])


# --------------------------------------------------------------------------- plain forms
def _turns(grid, d):
    """cos and sin (N, 1, pairs) of the rotation: d / 6 pairs for each axis, frequencies falling from 1."""
    p = d // 6
    freq = BASE ** (-torch.arange(p, dtype=torch.float64, device=grid.device) / p)
    angle = (grid.double()[:, :, None] * freq).reshape(grid.shape[0], 1, 3 * p)
    return angle.cos().float(), angle.sin().float()


def _rotate(x, cos, sin):
    """Neighbouring values of the first pairs turned, the others as they are."""
    m = 2 * cos.shape[-1]
    a, b = x[..., 0:m:2], x[..., 1:m:2]
    pairs = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([pairs, x[..., m:]], -1)


def _qk_plain(st, case):
    n, c, h = case["n"], case["channels"], case["heads"]
    d = c // h
    x = st["qkv"].float()
    cos, sin = _turns(st["grid"], d)
    normed, inv, outs = [], [], []
    for i, w in enumerate(st["weights"]):
        y = x[:, i * c:(i + 1) * c].reshape(n, h, d)
        inv.append((y.square().mean(-1, keepdim=True) + EPS).rsqrt())
        normed.append(y * inv[i])
        outs.append(_rotate(normed[i] * w.float(), cos, sin).reshape(n, c))
    out = torch.cat(outs + [x[:, 2 * c:]], 1).to(st["dtype"])
    if not case["train"]:
        return out
    dout, grads, dws = st["dout"].float(), [], []
    for i, w in enumerate(st["weights"]):
        dy = _rotate(dout[:, i * c:(i + 1) * c].reshape(n, h, d), cos, -sin)
        dws.append((dy * normed[i]).sum((0, 1)).to(st["dtype"]))
        dn = dy * w.float()
        grads.append((inv[i] * (dn - normed[i] * (dn * normed[i]).mean(-1, keepdim=True))).reshape(n, c))
    return out, torch.cat(grads + [dout[:, 2 * c:]], 1).to(st["dtype"]), dws[0], dws[1]


def _attention_plain(st, case):
    n, c, h = case["n"], case["channels"], case["heads"]
    maps = 2 if case["path"] == "diff" else 1
    w = c // h                                    # of a head's values
    d = w // maps                                 # of one map's queries and keys
    scale = d ** -0.5
    # sequences side by side, (S, L): the point of every row, which rows there are, the row that each point owns
    cu, L = st["cu"].long(), st["longest"]
    rows = cu[:-1, None] + torch.arange(L, device=cu.device)
    there = rows < cu[1:, None]
    S = rows.shape[0]
    point = st["order"][st["pad"][rows.clamp_max(st["pad"].shape[0] - 1)]]
    inverse = torch.empty_like(st["order"])
    inverse[st["order"]] = torch.arange(n, device=cu.device)
    owned = st["unpad"][inverse]
    seq = torch.searchsorted(cu, owned, right=True) - 1
    owned = seq * L + owned - cu[seq]

    x = st["qkv"][point].float()
    q = x[..., :c].reshape(S, L, h, maps, d).permute(0, 2, 3, 1, 4)
    k = x[..., c:2 * c].reshape(S, L, h, maps, d).permute(0, 2, 3, 1, 4)
    v = x[..., 2 * c:].reshape(S, L, h, w).transpose(1, 2)
    s = q @ k.transpose(-1, -2) * scale           # (S, h, maps, L, L)
    if case["path"] == "bias":
        grid, table = st["grid"][point].long(), st["table"].float()
        num = table.shape[0] // 3
        off = (grid[:, :, None] - grid[:, None]).clamp(-case["bound"], case["bound"]) + case["bound"]
        bucket = (off if st["buckets"] is None else st["buckets"].long()[off]) + num * torch.arange(3, device=cu.device)
        s = s + (table[bucket[..., 0]] + table[bucket[..., 1]] + table[bucket[..., 2]]).permute(0, 3, 1, 2)[:, :, None]
    s = s.masked_fill(~there[:, None, None, None, :], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    del s
    p = p / p.sum(-1, keepdim=True)
    if maps == 2:
        lam = st["lam"].float()[None, :, None, None]
        mix = p[:, :, 0] - lam * p[:, :, 1]
    else:
        mix = p[:, :, 0]
    out = (mix @ v).transpose(1, 2).reshape(S * L, c)[owned].to(st["dtype"])
    if not case["train"]:
        return out

    do = torch.zeros(S * L, c, device=cu.device)
    do[owned] = st["dout"].float()
    do = do.reshape(S, L, h, w).transpose(1, 2)
    dv = mix.transpose(-1, -2) @ do
    del mix
    dp = (do @ v.transpose(-1, -2))[:, :, None]
    mean = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - mean)
    del p, dp
    if maps == 2:
        dparam = -mean[:, :, 1].sum((0, 2, 3))
        ds[:, :, 1] *= -lam
    else:
        dparam = torch.zeros(3 * num, h, device=cu.device)
        for a in range(3):
            bins = torch.zeros(S, h, L, num, device=cu.device)
            bins.scatter_add_(3, (bucket[..., a] - a * num)[:, None].expand(-1, h, -1, -1), ds[:, :, 0])
            dparam[a * num:(a + 1) * num] = bins.sum((0, 2)).t()
        dparam = dparam.to(st["table"].dtype)
    dq = (ds @ k) * scale
    dk = (ds.transpose(-1, -2) @ q) * scale
    del ds
    dx = torch.cat([dq.permute(0, 3, 1, 2, 4).reshape(S, L, c), dk.permute(0, 3, 1, 2, 4).reshape(S, L, c),
                    dv.transpose(1, 2).reshape(S, L, c)], -1) * there[..., None]
    dqkv = torch.zeros(n, 3 * c, device=cu.device).index_add_(0, point.reshape(-1), dx.reshape(S * L, 3 * c))
    return out, dqkv.to(st["dtype"]), dparam


# --------------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    leaves = [st["qkv"]] + (st["weights"] if case["path"] == "qk" else
                            [st["table"] if case["path"] == "bias" else st["lam"]])
    leaves = [t.double().requires_grad_(case["train"]) for t in leaves]
    if case["path"] == "qk":
        out = _qk_exact(leaves, st["grid"], case)
        if not case["train"]:
            return out
        return (out.detach(),) + torch.autograd.grad(out, leaves, st["dout"].double())
    grads = [torch.zeros_like(t) for t in leaves]
    out = torch.zeros(case["n"], case["channels"], dtype=torch.float64, device="cuda")
    ends = st["cu"].tolist()
    owner = torch.full((ends[-1],), -1, dtype=torch.int64, device="cuda")
    owner[st["unpad"]] = st["order"]              # the point that a row answers for
    for a, b in zip(ends[:-1], ends[1:]):
        points, answers = st["order"][st["pad"][a:b]], owner[a:b]
        o = _sequence_exact(leaves, points, st, case)
        keep = answers >= 0
        out[answers[keep]] = o.detach()[keep]
        if case["train"]:
            seed_grad = torch.where(keep[:, None], st["dout"].double()[answers.clamp_min(0)], 0.0)
            for total, part in zip(grads, torch.autograd.grad(o, leaves, seed_grad)):
                total += part
    return (out, grads[0], grads[1]) if case["train"] else out


def _qk_exact(leaves, grid, case):
    qkv, wq, wk = leaves
    n, c, h = case["n"], case["channels"], case["heads"]
    d, p = c // h, c // h // 6
    x = qkv.reshape(n, 3, h, d)
    freq = torch.tensor([BASE ** (-i / p) for i in range(p)], dtype=torch.float64, device=grid.device)
    turn = torch.polar(torch.ones(n, 3 * p, dtype=torch.float64, device=grid.device),
                       torch.einsum("na,p->nap", grid.double(), freq).reshape(n, 3 * p))[:, None]
    parts = []
    for i, w in ((0, wq), (1, wk)):
        y = x[:, i] / torch.sqrt(torch.mean(x[:, i] ** 2, -1, keepdim=True) + EPS) * w
        z = torch.view_as_complex(y[..., :6 * p].reshape(n, h, 3 * p, 2).contiguous()) * turn
        parts.append(torch.cat([torch.view_as_real(z).reshape(n, h, 6 * p), y[..., 6 * p:]], -1).reshape(n, c))
    return torch.cat(parts + [x[:, 2].reshape(n, c)], 1)


def _sequence_exact(leaves, points, st, case):
    """Attention of one sequence: (rows, channels)."""
    qkv, param = leaves
    c, h = case["channels"], case["heads"]
    q, k, v = (t.reshape(len(points), h, c // h).transpose(0, 1) for t in qkv[points].split(c, 1))
    if case["path"] == "diff":
        d = c // h // 2
        maps = [torch.softmax(torch.einsum("hid,hjd->hij", q[..., m], k[..., m]) / math.sqrt(d), -1)
                for m in (slice(0, d), slice(d, 2 * d))]
        a = maps[0] - param[:, None, None] * maps[1]
    else:
        g, num = st["grid"][points].long(), param.shape[0] // 3
        s = torch.einsum("hid,hjd->hij", q, k) / math.sqrt(c // h)
        for axis in range(3):
            off = torch.clamp(g[:, None, axis] - g[None, :, axis], -case["bound"], case["bound"]) + case["bound"]
            if st["buckets"] is not None:
                off = st["buckets"].long()[off]
            s = s + torch.nn.functional.embedding(off, param[axis * num:(axis + 1) * num]).permute(2, 0, 1)
        a = torch.softmax(s, -1)
    return torch.einsum("hij,hjd->hid", a, v).transpose(0, 1).reshape(len(points), c)


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    n, c = case["n"], case["channels"]
    size = 4 if case["dtype"] == "fp32" else 2
    if case["path"] == "qk":
        rows = 4 if case["train"] else 2          # qkv and its result, gradients of both
        return {"bytes": float(n * (3 * c * size * rows + 12)), "flops": float(n * c * (60 if case["train"] else 20))}
    pairs = float(sum(v * v for v in _lengths(case)))
    rows = 8 if case["train"] else 4              # qkv and out, gradients of both
    index = 24 + (12 if case["path"] == "bias" else 0)
    flops = 4.0 * pairs * c                       # scores and values; three sums for each score's bias
    if case["path"] == "bias":
        flops += 3.0 * pairs * case["heads"]
    if case["train"]:
        flops += 10.0 * pairs * c
    return {"bytes": float(n * (c * size * rows + index)), "flops": flops}
