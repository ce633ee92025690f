"""Gradients and refusals of SerializedAttention and of a block around it by mode: training, evaluation, autograd on and off."""
import pytest
import torch

import pointtransformerv3_b200 as P
from helpers import rel_l2
from pointtransformerv3_b200 import _lib, ops
from test_attention_options_gpu import OPTIONS, module, reference, scene

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("name", [n for n in OPTIONS if n not in ("plain", "rpe")])
def test_gradients_in_evaluation(name, dtype):
    """A module with options beyond the reference's, frozen in evaluation mode: all gradients as in training mode, bit for bit, and
    without autograd none.  Bounds as for training: at most ten roundings of bf16, sums of fp32."""
    att = module(name, dtype, flash=True)
    pt, feat, dout = scene([300, 90], 51, 64, dtype)

    def run(training):
        att.train(training)
        x = feat.clone().requires_grad_()
        pt.feat = x
        out = att(pt).feat
        return (out.detach(),) + torch.autograd.grad(out, [x] + list(att.parameters()), dout)
    got = run(False)
    assert all(torch.equal(a, b) for a, b in zip(got, run(True)))
    want, _, dx = reference(att, pt, feat, dout)
    tol = 2e-5 if dtype == torch.float32 else 10 ** 0.5 * 2.0 ** -8
    assert rel_l2(got[0], want) < tol and rel_l2(got[1], dx) < tol
    att.eval()
    for p in att.parameters():
        p.requires_grad_(False)
    x = feat.clone().requires_grad_()                   # of the features alone
    pt.feat = x
    assert torch.equal(torch.autograd.grad(att(pt).feat, x, dout)[0], got[1])
    for p in att.parameters():
        p.requires_grad_(True)
    pt.feat = feat
    with torch.no_grad():
        out = att(pt).feat
    assert not out.requires_grad and rel_l2(out, want) < tol


def test_a_block_does_not_train_its_attention_alone():
    """Operators around the attention have no gradients, so a block in evaluation refuses an attention in training."""
    torch.manual_seed(0)
    block = P.Block(64, 4, 128, cpe_indice_key="s", upcast_attention=False, upcast_softmax=False,
                    attn_options=dict(qk_norm=True)).cuda().eval()
    pt, feat, _ = scene([200], 5, 64, torch.float32)
    pt.feat = feat
    pt.sparsify()
    with torch.no_grad():
        block(P.Point(dict(pt)))
    block.attn.train()
    with pytest.raises(AssertionError, match="inference only"):
        block(P.Point(dict(pt)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_a_bias_of_far_offsets_evaluates(dtype):
    """Patches of 10 000 have a bias for offsets up to 68, more than the inference kernel's table holds: what trains evaluates."""
    att = module("rpe", dtype, flash=False, K=10000)
    assert att.rpe.pos_bnd == 68
    pt, feat, dout = scene([300, 270], 61, 64, dtype)
    outs = []
    for training in (True, False):
        att.train(training)
        pt.feat = feat
        with torch.no_grad():
            outs.append(att(pt).feat)
    want = reference(att, pt, feat, dout)[0]
    for out in outs:
        assert rel_l2(out, want) < (2e-5 if dtype == torch.float32 else 10 ** 0.5 * 2.0 ** -8)


def test_what_does_not_hold_is_reported_in_training():
    """Coordinates that the bias does not take, by the call itself and without a look at the status word."""
    att = module("buckets", torch.float32, flash=False).train()
    pt, feat, _ = scene([200, 150], 71, 64, torch.float32)
    for bad in (True, False):
        q = P.Point(dict(pt))
        q["_status"] = ops.new_status("cuda")
        q.feat = feat
        if bad:
            q.grid_coord = pt.grid_coord.clone()
            q.grid_coord[7, 2] = 2 ** 22 + 1
            with pytest.raises(_lib.Ptv3Error, match="SerializedAttention.*index or size out of range"):
                att(q)
        else:
            att(q)


def test_a_captured_step_does_not_wait():
    """A Point that has not been reported on yet, in a step that is captured: forward and backward, replayed with other features."""
    att = module("all_diff", torch.bfloat16, flash=True).train()
    pt, feat, dout = scene([300, 100], 73, 64, torch.bfloat16)
    x = feat.clone().requires_grad_()

    def step(point):
        point.feat = x
        out = att(point).feat
        return (out,) + torch.autograd.grad(out, [x] + list(att.parameters()), dout)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(P.Point(dict(pt)))
    torch.cuda.current_stream().wait_stream(side)
    fresh = P.Point(dict(pt))
    att.get_padding_and_inverse(fresh)
    fresh.device_status()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(fresh)
    with torch.no_grad():
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(9)))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, step(P.Point(dict(pt)))))
    fresh.check_status(force=True)


def test_heads_without_gradients_evaluate_without_any():
    """Heads of 8 have norms and rotation and no gradients: refused in training, and in evaluation no part of the module has one."""
    att = module("norm_rope", torch.float32, flash=True, C=32, H=4)
    pt, feat, _ = scene([200, 90], 81, 32, torch.float32)
    outs = []
    for grad in (True, False):
        att.eval()
        pt.feat = feat.clone().requires_grad_()
        with torch.set_grad_enabled(grad):
            outs.append(att(pt).feat)
        assert not outs[-1].requires_grad
    assert torch.equal(*outs)
    pt.feat = feat
    with pytest.raises(ValueError, match="heads of 8"):
        att.train()(pt)
