"""Timed cases of what stands behind a network's logits: answers, losses and their gradients.

* ``score``: log probability of a label, entropy and the best alternatives of every point's logits
  (``functional.class_log_probs``); trained, it is the cross entropy's term and the entropy with their gradients;
* ``distill``: loss of a student's logits against a teacher's stored top classes (``functional.distill_topk``);
* ``head``: the answers of ``score`` straight from the features of a frozen network, its last Linear layer included
  (``ops.seg_head_log_probs``), as a teacher's lists are made.

Inputs are made on the GPU from the seed: logits of a network that has learnt most labels, with points left without a label and,
where a case says so, classes that a point's dataset does not have (minus infinity).  Numbers of points follow the levels of the
default backbone, numbers of classes go from a few over the long lists of open vocabularies to a codebook's.
"""
import math

import torch

own = False

IGNORE = -1           # label of a point without one
FAR = -1e5            # stands for minus infinity in 64 bits: its exponential is zero there


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # the points under a brush of an interactive tool: a call whose launch and host work are what counts
        dict(name="score_1k_20", path="score", train=False, n=1000, classes=20, top=3, labels=False, masked=False,
             temperature=1.0, dtype="bf16"),
        # validation of a batch of four rooms: loss, uncertainty and alternatives of every point
        dict(name="score_407k_20", path="score", train=False, n=407678, classes=20, top=5, labels=True, masked=False,
             temperature=1.0, dtype="bf16"),
        # a training step with two datasets of 200 classes in all, each point with the classes of its own
        dict(name="score_train_105k_200", path="score", train=True, n=105505, classes=200, top=0, labels=True, masked=True,
             temperature=1.0, dtype="bf16"),
        # fp32 training on a small indoor set of labels
        dict(name="score_train_64k_13_f32", path="score", train=True, n=64003, classes=13, top=0, labels=True, masked=False,
             temperature=1.0, dtype="fp32"),
        # pretraining against a codebook: the likeliest entries of masked patches
        dict(name="score_4k_8192_f32", path="score", train=False, n=4099, classes=8192, top=32, labels=True, masked=False,
             temperature=1.0, dtype="fp32"),
        # a student's step on the coarse level of one room
        dict(name="distill_train_1757_20", path="distill", train=True, n=1757, classes=20, top=4, rest=False, masked=False,
             temperature=2.0, dtype="bf16"),
        # a student's step on the benchmark's batch of rooms
        dict(name="distill_train_407k_20", path="distill", train=True, n=407678, classes=20, top=8, rest=True, masked=False,
             temperature=1.0, dtype="bf16"),
        # a student's step on a long list of classes, an odd number of them
        dict(name="distill_train_50k_1201", path="distill", train=True, n=50021, classes=1201, top=32, rest=False,
             masked=False, temperature=2.0, dtype="bf16"),
        # validation of a student in fp32
        dict(name="distill_30k_333_f32", path="distill", train=False, n=30011, classes=333, top=16, rest=True, masked=True,
             temperature=1.0, dtype="fp32"),
        # one room's third level, from features to answers
        dict(name="head_6k_64_20", path="head", train=False, n=6760, channels=64, classes=20, top=3, labels=False,
             temperature=1.0, dtype="bf16"),
        # a teacher's lists of the benchmark's batch of rooms
        dict(name="head_407k_64_20", path="head", train=False, n=407678, channels=64, classes=20, top=8, labels=True,
             temperature=1.0, dtype="bf16"),
        # a room scored against the embeddings of a long list of words
        dict(name="head_100k_512_1201", path="head", train=False, n=100003, channels=512, classes=1201, top=16, labels=True,
             temperature=2.0, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    path = rng.choice(("score", "score", "distill", "distill", "head"))
    temperature = rng.choice((1.0, 1.0, 2.0, 0.5, 3.0))
    if path == "head":
        channels, classes = 8 * rng.randint(2, 64), _log(rng, 2, 2000)
        n = _log(rng, 64, min(400000, 50000000000 // (channels * (classes + 64))))
        return dict(path=path, train=False, n=n, channels=channels, classes=classes, top=rng.choice((0, 1, 3, 8, 16, 32)),
                    labels=rng.random() < 0.5, temperature=temperature, dtype="bf16")
    classes = _log(rng, 2, 20000)
    n = _log(rng, 64, min(400000, 30000000 // classes))
    case = dict(path=path, train=rng.random() < 0.5, n=n, classes=classes, masked=classes > 8 and rng.random() < 0.4,
                temperature=temperature, dtype="fp32" if rng.random() < 0.3 else "bf16")
    # no list is longer than half the classes: those of one dataset of two
    longest = max(1, min(64, classes // 2))
    if path == "score":
        case.update(top=rng.choice((0, 1, rng.randint(1, longest))), labels=case["train"] or rng.random() < 0.6)
    else:
        case.update(top=rng.randint(1, longest), rest=rng.random() < 0.5)
    return case


# --------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = torch.float32 if case["dtype"] == "fp32" else torch.bfloat16
    n, k = case["n"], case["classes"]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    def uniform(*shape):
        return torch.rand(*shape, device="cuda", generator=g)
    st = dict(case=case, dtype=dtype, status=torch.zeros(1, dtype=torch.int32, device="cuda"), labels=None)
    label = torch.randint(0, k, (n, 1), device="cuda", generator=g)
    if case["path"] == "head":
        c = case["channels"]
        # steps of 1/16 and 1/256: sums of these are exact in 32 bits, so that the order of alternatives has one answer
        st["weight"] = ((normal(k, c) * (2 / math.sqrt(c)) * 256).round() / 256).clamp(-1, 1).to(dtype)
        st["bias"] = ((0.5 * normal(k) * 256).round() / 256).clamp(-0.5, 0.5).to(dtype)
        toward = 1.5 * st["weight"].float()[label[:, 0]]
        st["feat"] = (((normal(n, c) + toward) * 16).round() / 16).clamp(-4, 4).to(dtype)
    else:
        x = 1.5 * normal(n, k)
        x.scatter_add_(1, label, 3 + 2 * normal(n, 1))
        if case["masked"]:
            # two datasets: one has the classes of even numbers, the other those of odd ones
            other = (torch.arange(k, device="cuda")[None] - label) % 2 == 1
            x.masked_fill_(other, -math.inf)
        st["logits"] = x.to(dtype)
    if case["path"] == "distill":
        # a teacher of the same labels: its list of each point, a few points that it was not asked about
        teacher = 0.7 * x + 1.5 * normal(n, k)
        values, classes = (torch.log_softmax(teacher / case["temperature"], 1) if case["rest"] else teacher).topk(case["top"], 1)
        classes[uniform(n) < 0.03] = -1
        st["teacher"], st["classes"] = values, classes.int()
        if case["train"]:
            st["dout"] = 0.5 + uniform(n)
    elif case["labels"]:
        label = label[:, 0].clone()
        label[uniform(n) < 0.05] = IGNORE
        st["labels"] = label
        if case["train"]:
            # class weights of the cross entropy, and a small reward of certainty
            st["dout"] = -(0.5 + uniform(n)), 0.1 * uniform(n)
    return st


# --------------------------------------------------------------------------- one pass
def run(st):
    if own:
        return _run_own(st, st["case"])
    return _distill_plain(st, st["case"]) if st["case"]["path"] == "distill" else _score_plain(st, st["case"])


def _run_own(st, case):
    from pointtransformerv3_b200 import functional as F, ops
    if case["path"] == "head":
        return [t for t in ops.seg_head_log_probs(st["feat"], st["weight"], st["bias"], st["labels"], top=case["top"],
                                                  temperature=case["temperature"], status=st["status"]) if t is not None]
    x = st["logits"].detach().requires_grad_(case["train"])
    if case["path"] == "score":
        out = F.class_log_probs(x, st["labels"], top=case["top"], temperature=case["temperature"], status=st["status"])
        if case["train"]:
            dx = torch.autograd.grad((out.log_prob, out.entropy), x, st["dout"])
            return [t.detach() for t in out if t is not None] + [dx[0]]
        return [t for t in out if t is not None]
    loss = F.distill_topk(x, st["teacher"], st["classes"], temperature=case["temperature"], rest=case["rest"],
                          status=st["status"])
    if case["train"]:
        return [loss.detach(), torch.autograd.grad(loss, x, st["dout"])[0]]
    return [loss]


# --------------------------------------------------------------------------- plain forms
def _score_plain(st, case):
    if case["path"] == "head":
        x = st["feat"].float() @ st["weight"].float().t() + st["bias"].float()
    else:
        x = st["logits"].float()
    z = (x - x.amax(1, keepdim=True)) / case["temperature"]
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    logp = z - torch.log(total)
    p = e / total
    plogp = torch.where(p > 0, p * logp, 0.0)
    entropy = -plogp.sum(1)
    out = [entropy]
    if st["labels"] is not None:
        there = st["labels"] != IGNORE
        at = st["labels"].clamp_min(0)[:, None]
        out.insert(0, torch.where(there, logp.gather(1, at)[:, 0], 0.0))
    if case["top"]:
        k = min(case["top"], case["classes"])
        classes = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :k]
        values = logp.gather(1, classes)
        more = case["top"] - k
        out += [torch.nn.functional.pad(values, (0, more), value=-math.inf),
                torch.nn.functional.pad(classes, (0, more), value=-1).int()]
    if case["train"]:
        g, h = st["dout"][0] * there, st["dout"][1]
        dx = -p * g[:, None] - h[:, None] * (plogp + p * entropy[:, None])
        dx.scatter_add_(1, at, g[:, None])
        out.append((dx / case["temperature"]).to(st["dtype"]))
    return out


def _distill_plain(st, case):
    x, n = st["logits"].float(), case["n"]
    z = (x - x.amax(1, keepdim=True)) / case["temperature"]
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    logtotal = torch.log(total)
    there = st["classes"] >= 0
    at = st["classes"].long().clamp_min(0)
    v = st["teacher"].float().masked_fill(~there, -math.inf)
    if case["rest"]:
        t = torch.exp(v)
    else:
        t = torch.exp((v - v.amax(1, keepdim=True).clamp_min(-3e38)) / case["temperature"])
        t = t / t.sum(1, keepdim=True).clamp_min(1e-30)
    some = there.any(1)
    loss = torch.where(t > 0, t * (torch.log(t) - z.gather(1, at) + logtotal), 0.0).sum(1)
    mass = t.sum(1)
    if case["rest"]:
        left = (1 - t.double().sum(1)).clamp_min(0).float() * some
        # the classes outside the list; a class of a list has the number k there, a column of its own that is dropped
        inside = torch.zeros(n, case["classes"] + 1, dtype=torch.bool, device=x.device)
        inside.scatter_(1, torch.where(there, at, case["classes"]), True)
        outside = ~inside[:, :-1]
        zo = z.masked_fill(~outside, -math.inf)
        top = zo.amax(1, keepdim=True)
        eo = torch.exp(zo - top)
        logout = torch.log(eo.sum(1)) + top[:, 0]
        loss = loss + torch.where(left > 0, left * (torch.log(left) - logout + logtotal[:, 0]), 0.0)
        mass = mass + left
    if not case["train"]:
        return [loss]
    dx = mass[:, None] * (e / total)
    dx.scatter_add_(1, at, torch.where(there, -t, 0.0))
    if case["rest"]:
        dx = dx - left[:, None] * (eo / eo.sum(1, keepdim=True))
    return [loss, (dx * (st["dout"] / case["temperature"])[:, None]).to(st["dtype"])]


# --------------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    step = max(1, 2 ** 24 // case["classes"])          # points at a time
    parts = []
    for a in range(0, case["n"], step):
        rows = slice(a, a + step)
        if case["path"] == "head":
            x = torch.nn.functional.linear(st["feat"][rows].double(), st["weight"].double(), st["bias"].double())
        else:
            x = st["logits"][rows].double()
        x = torch.where(x == -math.inf, FAR, x).requires_grad_(case["train"])
        parts.append((_distill_exact if case["path"] == "distill" else _score_exact)(x, st, case, rows))
    return [torch.cat(p) for p in zip(*parts)]


def _score_exact(x, st, case, rows):
    logp = torch.log_softmax(x / case["temperature"], 1)
    entropy = -(torch.exp(logp) * logp).sum(1)
    out = [entropy.detach()]
    if st["labels"] is not None:
        # the ignored points' class is the first, counted zero times
        label = st["labels"][rows]
        one = torch.nn.functional.one_hot(label.clamp_min(0), case["classes"]) * (label != IGNORE)[:, None]
        picked = (logp * one).sum(1)
        out.insert(0, picked.detach())
    if case["top"]:
        k = min(case["top"], case["classes"])
        order = torch.argsort(-x.detach(), dim=1, stable=True)[:, :k]
        values, order = torch.take_along_dim(logp.detach(), order, 1), order.int()
        if case["top"] > k:
            fill = values.new_ones(len(values), case["top"] - k)
            values, order = torch.cat([values, fill * -math.inf], 1), torch.cat([order, -fill.int()], 1)
        out += [values, order]
    if case["train"]:
        g, h = (d[rows].double() for d in st["dout"])
        out += torch.autograd.grad((g * picked + h * entropy).sum(), x)
    return out


def _distill_exact(x, st, case, rows):
    z = x / case["temperature"]
    v, c = st["teacher"][rows].double(), st["classes"][rows].long()
    t = torch.exp(v) if case["rest"] else torch.softmax(v / case["temperature"], 1)
    t = t * (c >= 0)
    logp = torch.log_softmax(z, 1)
    loss = (torch.xlogy(t, t) - t * torch.take_along_dim(logp, c.clamp_min(0), 1)).sum(1)
    if case["rest"]:
        member = torch.zeros_like(x).scatter_reduce(1, c.clamp_min(0), (c >= 0).double(), "amax")
        left = torch.where((c >= 0).any(1), 1 - t.sum(1), 0.0).clamp_min(0)
        outside = torch.logsumexp(torch.where(member > 0, 2 * FAR, z), 1) - torch.logsumexp(z, 1)
        loss = loss + torch.xlogy(left, left) - left * outside
    if not case["train"]:
        return [loss]
    return [loss.detach()] + list(torch.autograd.grad((loss * st["dout"][rows].double()).sum(), x))


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    n, k, size = case["n"], case["classes"], 4 if case["dtype"] == "fp32" else 2
    pairs = float(n) * k
    if case["path"] == "distill":
        made = n * (case["top"] * 8 + 4 + (4 if case["train"] else 0))
    else:
        made = n * (4 + case["top"] * 8 + (12 if case["labels"] else 0) + (8 if case["train"] else 0))
    if case["path"] == "head":
        c = case["channels"]
        return {"bytes": float(made + (n * c + k * c + k) * size), "flops": pairs * (2 * c + 6)}
    return {"bytes": made + pairs * size * (2 if case["train"] else 1), "flops": pairs * (12 if case["train"] else 6)}
