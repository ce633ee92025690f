"""Bounds on the norm of what results and gradients of ``pointtransformerv3_b200.functional`` are off by, beside the elementwise ones of
functional_reference.py.

An elementwise bound adds up what every rounding could do at worst, which for a sum over many pairs (a table's gradient) is more than
the sum itself.  Roundings do not conspire, so the norm of the error stays near that of independent ones:

* bf16: probabilities, dS, the second map's result and what is stored are rounded to bf16, at most 2^-8 of a value each: four
  independent ones are 2 2^-8 of the norm at most, and a little more is allowed for;
* fp32: a score of W <= 64 products is off by about sqrt(64) half steps of 2^-24 times its size of up to six, 48 of them, which a
  probability has as its relative error; its exponential 4; sums over up to 1 024 rows sqrt(1 024) at most: 84 in all, 5e-6.

A gradient that is zero by its formula (a patch of one row) is what cancels.  fp32: a few half steps of dO V, which 2^-22 of the norm
of dO and the largest feature stands for.  bf16: dS is formed against an estimate of delta, dO times the stored result, which is off
by 2^-8 of it; the estimate's error is taken out exactly, but dS = P (G - estimate) is rounded to bf16 on the way, 2^-8 of a
difference that is itself 2^-8 of dO V: 2^-16.

A bf16 table's gradient is stored in bf16 whatever the features are: half a step, 2^-8 of each of its values, in fp32 beside the rest."""
import torch

TOLERANCE = {torch.bfloat16: 2.5 * 2.0 ** -8, torch.float32: 84 * 2.0 ** -24}
FLOOR = {torch.bfloat16: 2.0 ** -16, torch.float32: 2.0 ** -22}


def parts(name, value):
    """Queries', keys' and values' gradients apart: one of them does not hide what another is off by."""
    if name == "dqkv":
        c = value.shape[1] // 3
        return [("dq", value[:, :c]), ("dk", value[:, c:2 * c]), ("dv", value[:, 2 * c:])]
    return [(name, value)]


def errors(got, ref, name, qkv, dout, dtype):
    """[(part, error's norm, bound)]; ``dtype``: of the features, whose products the kernels form."""
    out = []
    tolerance = TOLERANCE[dtype]
    if got.dtype == torch.bfloat16 and dtype == torch.float32:
        tolerance += 2.0 ** -8
    floor = FLOOR[dtype] * float(dout.double().norm()) * float(qkv.double().abs().max())
    for (what, value), (_, g) in zip(parts(name, ref[name][0]), parts(name, got.double())):
        out.append((what, float((g - value).norm()), tolerance * float(value.norm()) + floor))
    return out


def check(got, ref, name, qkv, dout, dtype, what=""):
    for part, err, bound in errors(got, ref, name, qkv, dout, dtype):
        assert err <= bound, "%s %s: off by %g, bound %g" % (what, part, err, bound)
