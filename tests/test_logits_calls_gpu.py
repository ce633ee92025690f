"""The operators behind the logits as a training program calls them: checkpointed, with saved tensors kept elsewhere, timed, two graphs at once, the
same tensor as several arguments; and the transforms that they refuse.  All by comparison with the plain call, bit for bit."""
import pytest
import torch

from pointtransformerv3_b200 import ops
from pointtransformerv3_b200 import functional as F

pytestmark = pytest.mark.gpu

SIZES = [20, 200, 1500]


def normal(*shape, seed, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def operands(n, K, dtype=torch.bfloat16):
    """Logits (rows of wider ones), labels, a teacher's list."""
    g = torch.Generator().manual_seed(1)
    x = normal(n, K + 8, seed=2, dtype=dtype)[:, :K]
    labels = torch.randint(-1, K, (n,), generator=g).cuda()
    values, classes = normal(n, K, seed=3).log_softmax(1).topk(6)
    return x, labels, values, classes


def losses(x, labels, values, classes, status):
    out = F.class_log_probs(x, labels, 4, status=status)
    return out.log_prob, out.entropy, out.top_log_probs, F.distill_topk(x, values, classes, rest=True, status=status)


def total(x, *args):
    return sum(t.sum() for t in losses(x, *args))


def same(a, b):
    return all(torch.equal(s, t) for s, t in zip(a, b))


@pytest.mark.parametrize("K", SIZES)
def test_checkpointed_and_offloaded(K):
    x, *rest = operands(300, K)
    rest.append(ops.new_status("cuda"))
    leaf = x.detach().requires_grad_()
    want = torch.autograd.grad(total(leaf, *rest), leaf)[0]
    for reentrant in (False, True):
        leaf = x.detach().requires_grad_()
        loss = torch.utils.checkpoint.checkpoint(total, leaf, *rest, use_reentrant=reentrant)
        loss.backward()
        assert torch.equal(leaf.grad, want)
    leaf = x.detach().requires_grad_()
    with torch.autograd.graph.save_on_cpu():
        loss = total(leaf, *rest)
    assert torch.equal(torch.autograd.grad(loss, leaf, retain_graph=True)[0], want)
    assert torch.equal(torch.autograd.grad(loss, leaf)[0], want)          # a second time from the same graph
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(loss, leaf)


@pytest.mark.parametrize("K", SIZES)
def test_timed_calls(K, monkeypatch):
    x, labels, values, classes = operands(300, K)
    status = ops.new_status("cuda")
    feat, weight = normal(300, 64, seed=5, dtype=torch.bfloat16), normal(K, 64, seed=6, dtype=torch.bfloat16)

    def step():
        leaf = x.detach().requires_grad_()
        out = losses(leaf, labels, values, classes, status)
        with torch.no_grad():
            plain = losses(x, labels, values, classes, status)
        return [*out, *plain, *torch.autograd.grad(sum(t.sum() for t in out), leaf),
                *ops.seg_head_log_probs(feat, weight, None, labels, 4, status=status)]
    want = step()
    monkeypatch.setattr(ops, "TIMERS", {})
    got = step()
    assert same(got, want) and len(ops.TIMERS) >= 3


@pytest.mark.parametrize("K", SIZES)
def test_two_graphs_of_one_call(K):
    """Captured calls share no memory but their arguments: replayed in either order and both at once, each answers for its own input."""
    x, *rest = operands(300, K)
    rest.append(ops.new_status("cuda"))
    held = [x.clone(), normal(300, K, seed=7, dtype=x.dtype)]
    graphs, outs = [], []

    def step(x):
        leaf = x.detach().requires_grad_()
        out = losses(leaf, *rest)
        return [*(t.detach() for t in out), torch.autograd.grad(sum(t.sum() for t in out), leaf)[0]]
    for h in held:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(h))
        graphs.append(graph)
    wants = [step(h) for h in held]
    for order in ((0, 1), (1, 0)):
        for i in order:
            graphs[i].replay()
        assert all(same(o, w) for o, w in zip(outs, wants))
    sides = [torch.cuda.Stream() for _ in graphs]
    for side, graph in zip(sides, graphs):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph.replay()
    for side in sides:
        torch.cuda.current_stream().wait_stream(side)
    assert all(same(o, w) for o, w in zip(outs, wants))


@pytest.mark.parametrize("K", SIZES)
def test_a_student_against_its_own_values(K):
    """A list cut from the student's own logits: the same memory is the student's, which has a gradient, and the teacher's, which has none."""
    leaf = normal(300, K, seed=8).requires_grad_()
    classes = torch.arange(8, dtype=torch.int32, device="cuda").expand(300, 8)
    args = dict(temperature=2.0, status=ops.new_status("cuda"))
    got = F.distill_topk(leaf, leaf[:, :8].detach(), classes, **args)
    want = F.distill_topk(leaf, leaf[:, :8].detach().clone(), classes.clone(), **args)
    assert torch.equal(got, want)
    assert torch.equal(torch.autograd.grad(got.sum(), leaf)[0], torch.autograd.grad(want.sum(), leaf)[0])


def test_transforms_are_refused():
    x, labels, values, classes = operands(4, 20, torch.float32)
    status = ops.new_status("cuda")
    with pytest.raises(RuntimeError):
        torch.func.grad(total)(x, labels, values, classes, status)
    for f in (lambda x: F.class_log_probs(x, top=2).entropy, lambda x: F.distill_topk(x, values, classes, status=status)):
        with pytest.raises(RuntimeError):
            torch.func.vmap(f)(torch.stack([x, x]))
