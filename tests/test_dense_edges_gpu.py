"""The dense operators on inputs at the edges of their ranges.

u = 2^-24, half a step of fp32. The activation's value: exp2 and rcp of the
hardware are within a step (2 u each), expf within a step too; then come at most
the correction's product, the sum with 1, the quotient, the product with up and the
scale's division, 1 u each: 9 u in all, and 1 u more for a code's own quotient.
"""

import pytest
import torch
from test_dense_ops_gpu import _layer, _product_ref, _rand, _run_layer

import flaggems_sglang as fgs
from flaggems_sglang import testing
from oracle import moe_ref

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF16, F32 = torch.bfloat16, torch.float32


def _silu(g, u):
    g, u = g.double(), u.double()
    return g * torch.sigmoid(g) * u


@pytest.mark.parametrize("lo,hi,up", [(-20.0, 20.0, 3.0), (-86.9, 20.0, 1e15),
                                      (-100.0, -86.0, 1e34), (80.0, 200.0, 0.5)])
@pytest.mark.parametrize("kind", ["fp8", "int8"])
def test_scale_of_one_gate(gpu, lo, hi, up, kind):
    """Rows of one value, so a row's scale is its magnitude over the format's
    largest: the silu's own accuracy from deep negative gates to large ones."""
    g = torch.linspace(lo, hi, 30011)
    x = torch.stack([g, torch.full_like(g, up)], 1)
    top = 448 if kind == "fp8" else 127
    ref = _silu(x[:, 0], x[:, 1]).abs() / top
    for copies in (1, 8):  # one by one, and in whole vectors
        wide = x.repeat_interleave(copies, 1).contiguous().to(gpu)
        s = fgs.silu_and_mul_quant(wide, kind)[1].reshape(-1).double().cpu()
        seen = ref * top > 1e-9  # (below, the scale's lower bound)
        assert int(seen.sum()) > 15000
        off = (s - ref).abs()[seen] / ref[seen]
        assert off.max() <= 9 * U, f"{float(off.max()) / U} u"


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,n", [(999, 2560), (1500, 250), (2048, 512)])
def test_int8_codes_of_loud_channels(gpu, rows, n, dtype):
    """Gates and ups of a few loud channels and of rows of differing norms
    (gates to about 50): every code is the nearest to its value over the scale
    but for the value's own roundings."""
    gen = torch.Generator().manual_seed(rows + n)
    x = torch.randn(rows, 2 * n, generator=gen)
    x *= torch.where(torch.rand(2 * n, generator=gen) < 0.01, 8.0, 1.0)
    x *= 0.5 + torch.rand(rows, 1, generator=gen)
    x = x.to(dtype)
    q, s = fgs.silu_and_mul_quant(x.to(gpu), "int8")
    v = _silu(*x.chunk(2, -1))
    ref = v.abs().amax(-1).clamp(min=1e-10) / 127
    s = s.double().cpu()
    assert ((s - ref).abs() <= 9 * U * ref).all()
    t = v / s[:, None]
    off = (q.double().cpu() - t).abs() - (0.5 + 10 * U * t.abs())
    assert off.max() <= 0, float(off.max())


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("rows,n", [(300, 2560), (1500, 250), (4096, 6144)])
def test_codes_of_loud_channels(gpu, activation, rows, n):
    """As above to e4m3, and with the exact gelu: its erfc's argument, rounded in
    its constant and its product, moves a negative gate's value by 2 g^2 u, and
    erfc itself is taken to be within 64 u."""
    gen = torch.Generator().manual_seed(rows - n)
    x = torch.randn(rows, 2 * n, generator=gen)
    x *= torch.where(torch.rand(2 * n, generator=gen) < 0.01, 8.0, 1.0)
    x *= 0.5 + torch.rand(rows, 1, generator=gen)
    x = x.to(BF16)
    g, u = x.to(gpu).double().chunk(2, -1)
    if activation == "silu":
        v, rel = g * torch.sigmoid(g) * u, 10 * U
    else:
        v, rel = g * 0.5 * torch.erfc(-g / 2 ** 0.5) * u, (2 * g.clamp(max=0) ** 2 + 74) * U
    for kind in ("fp8", "int8"):
        q, s = fgs.silu_and_mul_quant(x.to(gpu), kind, activation=activation)
        s = s.double().reshape(rows, -1)
        t = v / s.repeat_interleave(128 if kind == "fp8" else n, 1)[:, :n]
        half = torch.full_like(t, 0.5) if kind == "int8" else (
            2.0 ** -4 * t.abs()).clamp(min=2.0 ** -10)
        off = (q.double() - t).abs() - (half + rel * t.abs())
        assert off.max() <= 0, float(off.max())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n", [256, 250])
def test_activation_of_infinite_gates(gpu, n, dtype):
    """A gate of +infinity gives infinity, one of -infinity NaN, as the
    formula's steps; finite ones beyond 87 their values, zero from about -200."""
    x = torch.ones(6, 2 * n)
    x[1, 5] = float("inf")
    x[2, 6] = -float("inf")
    x[3, 7], x[3, n + 7] = 300.0, -2.0
    x[4, :n] = -1000.0
    x[4, 8], x[4, 9] = float("nan"), 88.0
    x[5, :n] = -200.0
    x = x.to(dtype).to(gpu)
    q, s = fgs.silu_and_mul_quant(x)
    q, s = q.float().cpu(), s.cpu()
    assert s[1, 0].isinf() and q[1, 5].isnan() and (q[1, 6:128] == 0).all()
    assert s[2, 0].isnan() and not s[1:3, 1].isnan().any()
    assert s[3, 0] == torch.tensor(600.0) / 448 and q[3, 7] == -448
    assert s[4, 0].isnan() and (q[4, 128:] == 0).all()
    assert (q[5] == 0).all() and (s[5] == torch.tensor(1e-10) / 448).all()
    q, s = fgs.silu_and_mul_quant(x, "int8")
    q, s = q.cpu(), s.cpu()
    assert s[1].isinf() and s[2].isnan() and s[4].isnan() and (q[4] == 0).all()
    assert s[3] == torch.tensor(600.0) / 127 and q[3, 7] == -127


def test_tensors_that_cannot_be_taken(gpu):
    """Inside a transformation, with a tangent, without memory: an error each,
    before any launch; the process and the calls after them go on."""
    x = torch.ones(4, 256, dtype=BF16, device=gpu)
    w = torch.ones(256, dtype=BF16, device=gpu)
    first = fgs.fused_rms_norm(x, w, residual=x)
    calls = (lambda t: fgs.fused_rms_norm(t, w).norm, lambda t: fgs.silu_and_mul_quant(t)[1],
             lambda t: fgs.fused_rms_norm(x, w, residual=t).norm)
    for call in calls:
        with pytest.raises(RuntimeError, match="no storage"):
            torch.vmap(call)(torch.ones(3, 4, 256, dtype=BF16, device=gpu))
        with pytest.raises(RuntimeError, match="no storage|tangent"):
            torch.func.jvp(call, (x,), (x,))
        with torch.autograd.forward_ad.dual_level():
            dual = torch.autograd.forward_ad.make_dual(x, x)
            with pytest.raises(RuntimeError, match="tangent"):
                call(dual)
        freed = torch.ones(8, 256, dtype=BF16, device=gpu)[4:]
        freed.untyped_storage().resize_(0)
        with pytest.raises(RuntimeError, match="no memory"):
            call(freed)
    again = fgs.fused_rms_norm(x, w, residual=x)
    assert torch.equal(again.norm, first.norm) and torch.equal(again.residual, x + x)


def test_in_place_beside_its_input(gpu):
    """x and an in-place residual as columns of one wider tensor, and refusals
    where they overlap."""
    gen = torch.Generator().manual_seed(2)
    wide = torch.randn(37, 1024, generator=gen).to(BF16).to(gpu)
    w = torch.randn(512, generator=gen).to(BF16).to(gpu)
    x, r = wide[:, :512], wide[:, 512:]
    ref = fgs.fused_rms_norm(x.contiguous(), w, residual=r.contiguous(), quant="fp8")
    for bad in (wide[:, 256:768], wide[:, 1:513]):
        with pytest.raises(ValueError, match="share no part"):
            fgs.fused_rms_norm(x, w, residual=bad, inplace=True)
    with pytest.raises(ValueError, match="share no part"):
        fgs.fused_rms_norm(r[1:], w, residual=r[:36], inplace=True)
    got = fgs.fused_rms_norm(x, w, residual=r, quant="fp8", inplace=True)
    assert torch.equal(got.q.view(torch.uint8), ref.q.view(torch.uint8))
    assert torch.equal(r, ref.residual) and torch.equal(x, wide[:, :512])


@pytest.mark.parametrize("m", [1, 19, 300])
def test_layer_against_the_oracle(gpu, m):
    """Both halves of the layer's run: the routed experts, fed with the norm's
    16-bit output, against the oracle under the bounds of its own tests, and
    their sum with the 64-bit product of the shared expert (the product's bound,
    and half a step for the sum). The check sees experts mistaken for their
    neighbours (planted in the oracle)."""
    gen = torch.Generator().manual_seed(m + 5)
    w, topk = _layer(gen, gpu)
    x, residual = (_rand(gen, (m, 512), BF16, gpu) for _ in range(2))
    n, h, q, s, routed, shared, out = _run_layer(w, topk, x, residual)
    tw, ti = fgs.fused_topk(n.norm, n.norm.float() @ w["router"], topk)
    tol = testing.TOL["fp8"]

    def oracle(ids):
        ref, mag = moe_ref.fused_moe(n.norm, w["w13"], w["w2"], tw, ids, mode="fp8",
                                     w1_scale=w["w13_scale"], w2_scale=w["w2_scale"],
                                     return_mag=True)
        return ref, mag, *moe_ref.compare(routed, ref, tol["atol"], tol["rtol"], mag)

    ref, mag, ok, max_abs, mean_rel = oracle(ti)
    assert ok and mean_rel <= tol["mean_rel"], (max_abs, mean_rel)
    wrong = oracle((ti + 1) % w["w2"].shape[0])
    assert not wrong[2] and wrong[4] > tol["mean_rel"]
    dense, terms = _product_ref(q, s, w["s2"], w["s2_scale"])
    dense, terms = dense.cpu(), terms.cpu()
    sums = (16 + 2 * 2 + 2) * 2.0 ** -23 + 7 * 2.0 ** -13
    near = tol["atol"] + tol["rtol"] * mag.double() + 1.01 * sums * terms + 2.0 ** -8 * dense.abs()
    whole = ref.double() + dense
    off = (out.double().cpu() - whole).abs() - near - 2.0 ** -8 * (whole.abs() + near)
    assert off.max() <= 0, float(off.max())


@pytest.mark.parametrize("rows,n,dtype", [(11000, 6144, BF16), (10500, 6500, BF16),
                                          (5500, 14336, BF16), (5600, 6144, F32),
                                          (2100, 40000, BF16), (1100, 65535, BF16)])
def test_activation_of_inputs_past_the_cache(gpu, rows, n, dtype):
    """Wide rows of more than 256 MB take a workgroup each: the bits of the same
    rows a few hundred at a time."""
    gen = torch.Generator(device=gpu).manual_seed(rows)
    x = torch.randn(rows, 2 * n, device=gpu, dtype=dtype, generator=gen)
    assert x.nbytes > 256 << 20
    for activation in ("silu", "gelu"):
        q, s = fgs.silu_and_mul_quant(x, activation=activation, column_major_scales=True)
        for at in range(0, rows, 700):
            q2, s2 = fgs.silu_and_mul_quant(x[at:at + 700], activation=activation)
            assert torch.equal(q[at:at + 700].view(torch.uint8), q2.view(torch.uint8))
            assert torch.equal(s[at:at + 700], s2)
