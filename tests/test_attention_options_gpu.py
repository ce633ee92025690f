"""SerializedAttention with its options, in evaluation and in training, against 64-bit forms of the same composition
(functional_reference.py), and a backbone made of such modules."""
import pytest
import torch

import functional_reference as R
import pointtransformerv3_b200 as P
from helpers import rel_l2, small_batch
from pointtransformerv3_b200 import functional as F

pytestmark = pytest.mark.gpu

OPTIONS = {
    "plain": dict(),
    "norm": dict(qk_norm=True),
    "rope": dict(enable_rope=True),
    "norm_rope": dict(qk_norm=True, enable_rope=True, rope_base=50.0),
    "rpe": dict(enable_rpe=True),
    "buckets": dict(enable_rpe=True, rpe_bound=40, qk_norm=True),
    "diff": dict(differential=True, differential_init=0.7),
    "all_diff": dict(differential=True, qk_norm=True, enable_rope=True),
}


def module(name, dtype, flash, C=64, H=2, K=128):
    kw = dict(OPTIONS[name])
    torch.manual_seed(3)
    att = P.SerializedAttention(C, H, K, enable_flash=flash and "enable_rpe" not in kw, upcast_attention=False,
                                upcast_softmax=False, **kw)
    with torch.no_grad():
        for n, p in att.named_parameters():
            if n in ("q_norm", "k_norm", "lam"):
                p.mul_(1 + 0.2 * torch.randn_like(p))
            if n == "rpe.rpe_table":
                p.copy_(0.5 * torch.randn_like(p))
    return att.cuda().to(dtype)


def scene(sizes, seed, C, dtype):
    data = small_batch(sizes, seed=seed)
    pt = P.Point({k: v.cuda() for k, v in data.items()})
    pt.serialization(order=["hilbert"], shuffle_orders=False)
    g = torch.Generator().manual_seed(seed)
    n = pt.batch.shape[0]
    return pt, torch.randn(n, C, generator=g).to(dtype).cuda(), torch.randn(n, C, generator=g).to(dtype).cuda()


def reference(att, pt, feat, dout):
    """(result, {parameter: gradient}, gradient of feat) in 64 bits."""
    params = {n: p.detach().double().requires_grad_() for n, p in att.named_parameters()}
    x = feat.detach().double().requires_grad_()
    pad, unpad, cu = att.get_padding_and_inverse(pt)
    qkv = x @ params["qkv.weight"].t() + params["qkv.bias"]
    if att.q_norm is not None or att.enable_rope:
        qkv = R.qk_norm_rope(qkv, att.num_heads * att.maps, pt.grid_coord if att.enable_rope else None, params.get("q_norm"),
                             params.get("k_norm"), base=att.rope_base)
    rpe = att.rpe
    param = params.get("rpe.rpe_table", params.get("lam"))
    args = (pt.serialized_order[0], pad, unpad, cu, att.num_heads, att.scale, att.maps, None if param is None else param.detach(),
            pt.grid_coord, rpe.pos_bnd if rpe is not None else 0, rpe.buckets if rpe is not None else None)
    core = R.attention(qkv.detach(), *args)["out"][0].requires_grad_()
    out = core @ params["proj.weight"].t() + params["proj.bias"]
    grads = dict(zip(("proj.weight", "proj.bias", "core"),
                     torch.autograd.grad(out, (params["proj.weight"], params["proj.bias"], core), dout.double())))
    res = R.attention(qkv.detach(), *args, grads.pop("core"))
    if param is not None:
        grads["rpe.rpe_table" if rpe is not None else "lam"] = res["dparam"][0]
    rest = [n for n in params if n not in grads]
    got = torch.autograd.grad(qkv, [params[n] for n in rest] + [x], res["dqkv"][0])
    grads.update(zip(rest, got))
    return out.detach(), grads, got[-1]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("name", list(OPTIONS))
def test_module_trains(name, dtype):
    """Results and gradients of the whole module.  In bf16 they pass through at most ten roundings one behind the other (qkv,
    norms, probabilities, core, projection, and back), each off by half a step, 2^-8 of a value, to all sides; in fp32 sums
    of 64 products and of patches of 128 rows."""
    att = module(name, dtype, flash=True).train()
    pt, feat, dout = scene([700, 90, 300], 31, 64, dtype)
    x = feat.clone().requires_grad_()
    pt.feat = x
    out = att(pt).feat
    grads = torch.autograd.grad(out, [x] + list(att.parameters()), dout)
    want, dparams, dx = reference(att, pt, feat, dout)
    tol = 2e-5 if dtype == torch.float32 else 10 ** 0.5 * 2.0 ** -8
    assert rel_l2(out.detach(), want) < tol
    assert rel_l2(grads[0], dx) < tol, "features"
    for (n, _), g in zip(att.named_parameters(), grads[1:]):
        # (of the key's bias only rounding is left without a norm: it shifts a row's scores alike)
        if n == "qkv.bias" and att.k_norm is None:
            C = g.shape[0] // 3
            keep = torch.cat([torch.arange(C), torch.arange(2 * C, 3 * C)]).cuda()
            assert rel_l2(g[keep], dparams[n][keep]) < tol, n
        else:
            assert rel_l2(g, dparams[n]) < tol, n
    pt.check_status(force=True)


@pytest.mark.parametrize("flash", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("name", list(OPTIONS))
def test_module_evaluates(name, dtype, flash):
    """The same result in evaluation, whichever kernels that takes, the core without a graph, and in inference mode."""
    att = module(name, dtype, flash).eval()
    pt, feat, dout = scene([500, 260], 33, 64, dtype)
    pt.feat = feat
    with torch.inference_mode():
        out = att(pt).feat
    want, _, _ = reference(att, pt, feat, dout)
    assert rel_l2(out, want) < (2e-5 if dtype == torch.float32 else 10 ** 0.5 * 2.0 ** -8)
    # (the Linear layers in fp32 are torch's and have their graph where the caller leaves it on; the core has none)
    assert not att.core(pt, torch.cat([feat] * 3, 1)).requires_grad
    att.train()
    pt.feat = feat
    assert rel_l2(att(pt).feat.detach(), want) < (2e-5 if dtype == torch.float32 else 10 ** 0.5 * 2.0 ** -8)


def test_a_step_lowers_what_its_gradient_says():
    """A small step against the gradient of all parameters changes the loss by about its square, to first order."""
    att = module("all_diff", torch.float32, True).train()
    pt, feat, dout = scene([400, 50], 35, 64, torch.float32)

    def loss():
        pt.feat = feat
        return (att(pt).feat.double() * dout.double()).sum()
    grads = torch.autograd.grad(loss(), list(att.parameters()))
    square = sum(float(g.double().square().sum()) for g in grads)
    ends = []
    step = 1e-3 / square ** 0.5
    with torch.no_grad():
        for sign in (1, -2):
            for p, g in zip(att.parameters(), grads):
                p.add_(sign * step * g)
            ends.append(float(loss()))
    # results off by 2^-20 of their size, 450 x 64 of them of about one, over a way of 2e-3; and a third derivative's 1e-6
    assert abs((ends[0] - ends[1]) / (2 * step) - square) < 0.02 * square


def test_rpe_module_with_buckets_in_tensor_form():
    """RPE.forward, the tensor form, against the bias that the kernel adds."""
    rpe = P.RPE(128, 3, bound=30).cuda()
    coord = torch.randint(-60, 60, (2, 5, 5, 3), device="cuda")
    got = rpe(coord)
    zero = torch.zeros(1, 3, dtype=torch.int64, device="cuda")
    want = R.bias_of(rpe.rpe_table.double(), coord.reshape(-1, 3), zero, 30, rpe.buckets)[:, :, 0].reshape(3, 2, 5, 5)
    assert torch.allclose(got.double(), want.permute(1, 0, 2, 3), atol=1e-6)


@pytest.mark.parametrize("name", ["norm_rope", "buckets", "all_diff"])
def test_backbone_of_such_modules(name):
    """A network whose attention has the options: bf16 near its fp32, the same bits on every pass, and no other network's
    results changed by it."""
    cfg = dict(enc_depths=(1, 1, 1), enc_channels=(32, 64, 64), enc_num_head=(2, 4, 4), enc_patch_size=(128,) * 3,
               dec_depths=(1, 1), dec_channels=(32, 64), dec_num_head=(2, 4), dec_patch_size=(128,) * 2, stride=(2, 2))
    opts = dict(OPTIONS[name])
    rpe = opts.pop("enable_rpe", False)
    if opts.get("differential"):
        cfg.update(enc_num_head=(1, 2, 2), dec_num_head=(1, 2))
    data = small_batch([900, 350], seed=41)
    torch.manual_seed(0)
    net = P.PointTransformerV3(in_channels=6, enable_flash=not rpe, enable_rpe=rpe, shuffle_orders=False, attn_options=opts,
                               **cfg).eval().cuda()
    outs = {}
    for dtype in (torch.float32, torch.bfloat16):
        net = net.to(dtype)
        runs = []
        for _ in range(2):
            d = {k: v.cuda() for k, v in data.items()}
            d["feat"] = d["feat"].to(dtype)
            torch.manual_seed(1)           # (poolings draw their orders from torch's generator)
            with torch.inference_mode():
                runs.append(net(d).feat)
        assert torch.equal(runs[0], runs[1])
        outs[dtype] = runs[0]
    assert bool(torch.isfinite(outs[torch.float32]).all())
    # bf16 through six blocks: each a chain of roundings as in test_module_trains, added up over the residual sums
    assert rel_l2(outs[torch.bfloat16], outs[torch.float32]) < 6 ** 0.5 * 10 ** 0.5 * 2.0 ** -8


def test_refused_options():
    with pytest.raises(AssertionError):
        P.SerializedAttention(32, 2, 64, enable_rpe=True, enable_flash=False, differential=True)
    with pytest.raises(AssertionError):
        P.SerializedAttention(32, 2, 64, enable_flash=False, rpe_bound=20)
    pt, feat, _ = scene([100], 1, 32, torch.float32)
    pt.feat = feat
    with pytest.raises(AssertionError):
        P.SerializedAttention(32, 2, 64, attn_drop=0.1, enable_flash=False).cuda().train()(pt)
    with pytest.raises(ValueError, match="heads of 8"):
        P.SerializedAttention(32, 4, 64, enable_flash=False).cuda().train()(pt)
    assert F.log_buckets(40)[1] == P.RPE(64, 2, bound=40).rpe_num
