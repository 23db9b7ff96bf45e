"""The bias's gradient through an activation: a sum of values that are rounded once, at
its end."""

import pytest
import torch

import flaggems_sglang as fgs
import steps_ref as ref
from test_linear_gpu import TYPES, inputs

pytestmark = pytest.mark.gpu


def dbias(x, w, bias, dout, kind, gated):
    """(value, bound). dv is off by its fp32 steps (the slope's where |act''| takes v's
    own error, 2^-16 of exp and its like) and by the rounding, in bf16, of what its own
    rounding leaves: 2^-8 h of dv, and 2^-134 where that is less than bf16's smallest step.
    A sum of n terms is off by 2^-24 of their magnitudes n times over, and is rounded
    once."""
    h, fn = ref.half(x.dtype), 0.0 if kind == "relu" else 2.0 ** -16
    x, w, d = x.double(), w.double(), dout.double()
    n = w.shape[0] // (2 if gated else 1)
    v = x @ w.t() + bias.double()
    ev = (x.shape[1] + 2) * ref.F32 * (x.abs() @ w.abs().t() + bias.double().abs())
    a, slope = ref.act(v[:, :n], kind)
    curve = ref.CURVE[kind]
    if gated:
        u, eg, eu = v[:, n:], ev[:, :n], ev[:, n:]
        dv = torch.cat([d * u * slope, d * a], 1)
        e = torch.cat([d.abs() * (eu * (ref.SLOPE + curve * eg) + u.abs() * (curve * eg + fn * ref.SLOPE)),
                       d.abs() * (ref.SLOPE * eg + fn * (a.abs() + 1))], 1)
    else:
        dv = d * slope
        e = d.abs() * (curve * ev + fn * ref.SLOPE)
    e = e + 4 * ref.F32 * dv.abs()  # (the products of dv)
    e = e + 2.0 ** -8 * h * (dv.abs() + e) + 2.0 ** -134
    rows = dv.shape[0]
    value = dv.sum(0)
    bound = e.sum(0) + (rows + 1) * ref.F32 * (dv.abs() + e).sum(0)
    return value, bound + h * (value.abs() + bound) + ref.tiny(x, h)


CASES = [("relu", False), ("silu", False), ("gelu", False), ("silu", True), ("gelu", True), ("relu", True)]


@pytest.mark.parametrize("kind, gated", CASES)
@pytest.mark.parametrize("rows, n, k", [(64, 136, 72), (333, 264, 136), (4000, 64, 40)])
@pytest.mark.parametrize("dtype", TYPES)
def test_dense(gpu, dtype, rows, n, k, kind, gated):
    """Columns whose terms cancel: alternating signs of dout."""
    t, dout = inputs(rows, n, k, TYPES[dtype], gated, True, False)
    dout = dout.abs() * torch.tensor([1.0, -1.0], device="cuda", dtype=dout.dtype).repeat(rows)[:rows, None]
    if kind == "relu":  # (not at its corner, where an error of v takes the other slope)
        v = t["x"].double() @ t["w"].double().t() + t["bias"].double()
        dout = torch.where(v[:, :n].abs() < 1e-3, 0, dout)
    b = t["bias"].clone().requires_grad_()
    out = fgs.fused_linear(t["x"], t["w"], b, activation=kind, gated=gated)
    got, = torch.autograd.grad(out, b, dout)
    ref.close("dbias", got, *dbias(t["x"], t["w"], t["bias"], dout, kind, gated))


@pytest.mark.parametrize("dtype", TYPES)
def test_groups(gpu, dtype):
    counts = [300, 0, 1, 129, 70]
    rows, n, k = 520, 136, 72  # 20 behind
    t, dout = inputs(rows, n, k, TYPES[dtype], True, True, False, groups=5)
    dout[500:] = float("nan")
    leaves = {key: t[key].clone().requires_grad_() for key in ("x", "w", "bias")}
    out = fgs.grouped_linear(leaves["x"], leaves["w"], torch.tensor(counts, dtype=torch.int32, device="cuda"),
                             leaves["bias"], activation="silu", gated=True)
    got = torch.autograd.grad(out, list(leaves.values()), dout)[2]
    at = 0
    for e, c in enumerate(counts):
        s = slice(at, at + c)
        at += c
        ref.close("dbias", got[e], *dbias(t["x"][s], t["w"][e], t["bias"][e], dout[s], "silu", True))


def test_values_past_the_type(gpu):
    """fp16: a dv that is infinite in dz makes an infinite sum; no NaN."""
    x = torch.zeros(40, 64, dtype=torch.float16, device="cuda")
    w = torch.zeros(32, 64, dtype=torch.float16, device="cuda")
    b = torch.full((32,), 2.0, dtype=torch.float16, device="cuda", requires_grad=True)
    out = fgs.fused_linear(x, w, b, activation="silu")
    dout = torch.zeros(40, 32, dtype=torch.float16, device="cuda")
    dout[3] = 65504.0
    got, = torch.autograd.grad(out, b, dout)
    assert bool(got.isposinf().all())
