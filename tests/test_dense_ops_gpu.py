"""The dense operators around the routed experts against their definitions in
64 bits: the norm with residual and 8-bit output, the gated activation with an
8-bit output, and the block-scaled e4m3 product.

Tolerances. u = 2^-24. A row's sum of squares adds at most 64 terms a thread
and 22 in the trees, all positive, so it is within 90 u of the exact one and
1 / sqrt within 50 u; sums, products and the scale's division add a few more:
values and scales are held to REL = 2^-17 = 128 u, plus half a step of the
type where they are rounded (2^-8 bf16, 2^-11 fp16, 2^-24 fp32) and the
type's smallest subnormal. The activation: exp's argument and erfc's are
rounded once, which at |gate| <= 6 (the normal samples used stay below) moves
exp by 9 u and erfc by 2 x^2 = 36 u; with their own ulps inside REL. Codes: at most half a step of the
format from value / scale (e4m3: 2^-4 of the value, 2^-10 below 2^-6; int8:
1/2), plus REL of the value.
The product: the matrix instruction cuts each of eight neighbouring products
13 bits below the largest of them (seven cuts of 2^-13 of it at most); the sum
of the 16 groups of a block and the sum over blocks are at most 16 + 2 kb + 2
roundings of 2^-23 (a truncating adder's) of the terms' magnitude. Operands
whose products span at most 13 bits (exponents in a window of four, so product
exponents in one of seven, and six fraction bits) are not cut at all: with them
the roundings alone are the bound.
"""

import threading

import pytest
import torch

import flaggems_sglang as fgs
from flaggems_sglang import _capi, quant

pytestmark = pytest.mark.gpu

REL = 2.0 ** -17
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -126}
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
FP8 = torch.float8_e4m3fn


def _near(got, ref, half, tiny=0.0):
    got, ref = got.double().cpu(), ref.double().cpu()
    assert got.shape == ref.shape
    off = (got - ref).abs() - ((half + REL) * ref.abs() + tiny)
    assert not (off > 0).any(), f"{float(off.max())} over the bound"
    assert not got.isnan().any()


def _check_codes(q, scales, v, kind):
    """Codes and scales of v (64 bits, [rows, cols])."""
    v = v.cpu()
    rows, cols = v.shape
    if kind == "int8":
        assert q.dtype == torch.int8
        ref = v.abs().amax(-1).clamp(min=1e-10) / 127
        _near(scales.reshape(rows), ref, HALF[F32])
        t = v / scales.reshape(rows, 1).double().cpu()
        off = (q.reshape(rows, cols).cpu().double() - t).abs() - (0.5 + REL * t.abs())
    else:
        assert q.dtype == FP8
        groups = -(-cols // 128)
        ref = torch.stack([v[:, 128 * g:128 * g + 128].abs().amax(-1) for g in range(groups)], 1)
        _near(scales.reshape(rows, groups), ref.clamp(min=1e-10) / 448, HALF[F32])
        s = scales.reshape(rows, groups).double().cpu().repeat_interleave(128, 1)[:, :cols]
        t = v / s
        step = torch.maximum(2.0 ** -4 * t.abs(), torch.tensor(2.0 ** -10, dtype=torch.float64))
        off = (q.reshape(rows, cols).cpu().double() - t).abs() - (step + REL * t.abs())
    assert not (off > 0).any(), f"code {float(off.max())} over the bound"


def _rand(gen, shape, dtype, device, loud=True):
    x = torch.randn(shape, generator=gen)
    if loud:
        x = x * torch.where(torch.rand(shape[-1], generator=gen) < 0.02, 8.0, 1.0)
    return x.to(dtype).to(device)


# ------------------------------------------------------------------- norm ---
def _norm_ref(x, weight, eps, residual, offset):
    h = x.double()
    if residual is not None:
        h = h + residual.double()
    n = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * (weight.double() + offset)
    return h, n


# rows and columns: one token, a wave a row and a workgroup a row, one to
# eight vectors a thread, tails inside a vector and inside a group
NORM_SHAPES = [(1, 7168), (1, 8), (1, 1), (3, 128), (5, 136), (2, 2048), (7, 200), (4, 100),
               (1025, 64), (1030, 512), (1027, 1000), (1024, 2048), (600, 4096), (513, 7168),
               (2, 16384), (3, 40000), (1, 65536), (9, 129), (2, 4099), (515, 1001)]


@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
@pytest.mark.parametrize("kind", [None, "fp8", "int8"])
def test_norm(gpu, rows, cols, kind):
    gen = torch.Generator().manual_seed(rows * 7 + cols)
    for dtype, wdtype, res in ((BF16, BF16, True), (F16, F32, False), (F32, F32, True),
                               (BF16, F32, False)):
        x = _rand(gen, (rows, cols), dtype, gpu)
        w = (1 + 0.1 * torch.randn(cols, generator=gen)).to(wdtype).to(gpu)
        r = _rand(gen, (rows, cols), dtype, gpu) if res else None
        offset = 0.0 if res else 1.0
        o = fgs.fused_rms_norm(x, w, 1e-5, r, weight_offset=offset, quant=kind, return_norm=True)
        h, n = _norm_ref(x, w, 1e-5, r, offset)
        _near(o.norm, n, HALF[dtype], TINY[dtype])
        assert (o.residual is None) == (r is None)
        if res:
            _near(o.residual, h, HALF[dtype], TINY[dtype])
        if kind:
            _check_codes(o.q, o.scales, n, kind)
        else:
            assert o.q is None and o.scales is None


@pytest.mark.parametrize("cols", [128, 1000, 7168])
def test_norm_outputs_do_not_depend_on_which_are_asked(gpu, cols):
    gen = torch.Generator().manual_seed(cols)
    x, r = (_rand(gen, (33, cols), BF16, gpu) for _ in range(2))
    w = _rand(gen, (cols,), BF16, gpu, loud=False)
    full = fgs.fused_rms_norm(x, w, 1e-6, r, quant="fp8", return_norm=True)
    plain = fgs.fused_rms_norm(x, w, 1e-6, r)
    only = fgs.fused_rms_norm(x, w, 1e-6, r, quant="fp8", column_major_scales=True)
    assert torch.equal(full.norm, plain.norm) and torch.equal(full.residual, plain.residual)
    assert only.norm is None and plain.q is None
    assert torch.equal(full.q.view(torch.uint8), only.q.view(torch.uint8))
    assert torch.equal(full.scales, only.scales)
    assert only.scales.stride() == (1, 33) and full.scales.is_contiguous()
    # in place, and x itself as the residual
    keep = r.clone()
    o = fgs.fused_rms_norm(x, w, 1e-6, keep, inplace=True)
    assert o.residual is keep
    assert torch.equal(keep, full.residual) and torch.equal(o.norm, full.norm)
    both = x.clone()
    o = fgs.fused_rms_norm(both, w, 1e-6, both, inplace=True)
    assert torch.equal(both, x + x)


@pytest.mark.parametrize("gap,start", [(64, 0), (8, 8), (3, 0), (1, 5)])
@pytest.mark.parametrize("kind", ["fp8", "int8"])
def test_norm_of_slices(gpu, gap, start, kind):
    """Rows of a wider tensor, aligned and not; the values around an in-place
    residual stay."""
    gen = torch.Generator().manual_seed(gap + start)
    rows, cols = 37, 512
    wide = _rand(gen, (rows, cols + gap + start), BF16, gpu)
    x = wide[:, start:start + cols]
    res = _rand(gen, (rows, cols + gap + start), BF16, gpu)
    before = res.clone()
    r = res[:, start:start + cols]
    w = _rand(gen, (cols,), BF16, gpu, loud=False)
    ref = fgs.fused_rms_norm(x.contiguous(), w, 1e-6, r.contiguous(), quant=kind, return_norm=True)
    o = fgs.fused_rms_norm(x, w, 1e-6, r, quant=kind, return_norm=True, inplace=True)
    assert torch.equal(o.norm, ref.norm) and torch.equal(o.scales, ref.scales)
    assert torch.equal(o.q.view(torch.uint8), ref.q.view(torch.uint8))
    assert torch.equal(res[:, start:start + cols], ref.residual)
    assert torch.equal(res[:, :start], before[:, :start])
    assert torch.equal(res[:, start + cols:], before[:, start + cols:])


def test_norm_of_more_dimensions_and_none(gpu):
    gen = torch.Generator().manual_seed(5)
    x = _rand(gen, (3, 5, 256), F16, gpu)
    w = _rand(gen, (256,), F16, gpu, loud=False)
    o = fgs.fused_rms_norm(x, w, quant="fp8", return_norm=True, column_major_scales=True)
    flat = fgs.fused_rms_norm(x.view(15, 256), w, quant="fp8", return_norm=True)
    assert o.norm.shape == x.shape and o.q.shape == x.shape and o.scales.shape == (3, 5, 2)
    assert torch.equal(o.norm.view(15, 256), flat.norm)
    assert torch.equal(o.scales.reshape(15, 2), flat.scales)
    swapped = fgs.fused_rms_norm(x.transpose(0, 1), w)
    assert torch.equal(swapped.norm, flat.norm.view(3, 5, 256).transpose(0, 1))
    one = fgs.fused_rms_norm(x[0, 0], w, quant="int8")
    assert one.q.shape == (256,) and one.scales.shape == ()
    empty = fgs.fused_rms_norm(x[:0], w, residual=x[:0], quant="fp8", return_norm=True)
    assert empty.norm.shape == (0, 5, 256) and empty.scales.shape == (0, 5, 2)
    assert empty.residual.shape == (0, 5, 256)


@pytest.mark.parametrize("cols", [256, 250, 2048])
def test_norm_of_zeros_nans_and_infinities(gpu, cols):
    x = torch.ones(6, cols)
    x[0] = 0.0
    x[1, 3] = float("nan")
    x[2, 200] = float("inf")
    x[3, 4] = -float("inf")
    x[4] = 1e-30
    w = torch.ones(cols, dtype=F32, device=gpu)
    for kind in ("fp8", "int8"):
        o = fgs.fused_rms_norm(x.to(gpu), w, 1e-6, quant=kind, return_norm=True)
        n = o.norm.cpu()
        assert (n[0] == 0).all() and (o.q[0].cpu().float() == 0).all()
        assert n[1].isnan().all()
        assert n[2, 200].isnan() and (n[2, :200] == 0).all()
        assert n[3, 4].isnan() and (n[3, 5:] == 0).all()
        assert (n[5] - 1).abs().max() < 1e-5
        s = o.scales.cpu()
        if kind == "int8":
            assert s[1:4].isnan().all() and s[0] > 0 and s[5] > 0
            assert (o.q[1:4].cpu() == 0).all()
        else:
            assert s[1].isnan().all() and s[2, 1].isnan() and s[3, 0].isnan()
            assert s[2, 0] > 0 and s[3, 1] > 0
            q = o.q.cpu().float()
            assert q[1].isnan().all() and q[2, 128:256].isnan().all() and (q[2, :128] == 0).all()


# -------------------------------------------------------------- activation ---
ACT_SHAPES = [(1, 2048), (8, 2048), (1, 1), (3, 100), (5, 136), (1025, 64), (1024, 1000),
              (1026, 768), (600, 2560), (2, 14336), (513, 7168), (1, 65536), (7, 4099),
              (1030, 512), (4096, 6144), (4097, 6500), (3, 40000)]


def _act_ref(x, gelu):
    g, u = x.double().cpu().chunk(2, -1)
    return (g * 0.5 * torch.erfc(-g / 2 ** 0.5) if gelu else g * torch.sigmoid(g)) * u


@pytest.mark.parametrize("rows,n", ACT_SHAPES)
@pytest.mark.parametrize("kind", ["fp8", "int8"])
def test_activation(gpu, rows, n, kind):
    gen = torch.Generator().manual_seed(rows * 3 + n)
    for dtype, gelu in ((BF16, False), (F16, True), (F32, False)):
        x = _rand(gen, (rows, 2 * n), dtype, gpu, loud=False)
        q, s = fgs.silu_and_mul_quant(x, kind, activation="gelu" if gelu else "silu")
        v = _act_ref(x, gelu)
        _check_codes(q, s, v, kind)
        if kind == "fp8":
            q2, s2 = fgs.silu_and_mul_quant(x, kind, activation="gelu" if gelu else "silu",
                                            column_major_scales=True)
            assert torch.equal(s, s2) and torch.equal(q.view(torch.uint8), q2.view(torch.uint8))
            assert s2.stride() == (1, rows) or rows == 1 or s2.shape[1] == 1


def test_activation_of_slices_and_none(gpu):
    gen = torch.Generator().manual_seed(9)
    wide = _rand(gen, (21, 1300), BF16, gpu)
    for a, b in ((0, 512), (8, 1288), (3, 1003)):
        q, s = fgs.silu_and_mul_quant(wide[:, a:b])
        q2, s2 = fgs.silu_and_mul_quant(wide[:, a:b].contiguous())
        assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s, s2)
    q, s = fgs.silu_and_mul_quant(wide[:0], "int8")
    assert q.shape == (0, 650) and s.shape == (0,)
    q, s = fgs.silu_and_mul_quant(wide.view(3, 7, 1300))
    assert q.shape == (3, 7, 650) and s.shape == (3, 7, 6)


@pytest.mark.parametrize("n", [256, 250])
def test_activation_of_nans_and_infinities(gpu, n):
    x = torch.ones(4, 2 * n)
    x[1, 5] = float("nan")
    x[2, n + 5] = float("inf")
    x[3, 7] = -float("inf")
    q, s = fgs.silu_and_mul_quant(x.to(gpu))
    q, s = q.cpu().float(), s.cpu()
    assert s[1, 0].isnan() and s[1, 1] > 0 and q[1, :128].isnan().all()
    assert s[2, 0].isinf() and q[2, 5].isnan() and (q[2, 6:128] == 0).all()
    assert s[3, 0].isnan()
    q, s = fgs.silu_and_mul_quant(x.to(gpu), "int8")
    assert s[1].isnan() and s[2].isinf() and (q[1:3].cpu() == 0).all()


# ----------------------------------------------------------------- product ---
def _operands(gen, m, n, k, device, narrow=False):
    """Random codes over the whole e4m3 range without NaN (narrow: magnitudes
    1 to 15), scales over four octaves."""
    def codes(rows):
        if narrow:
            c = torch.randint(0x38, 0x58, (rows, k), generator=gen, dtype=torch.uint8)
            c |= torch.randint(0, 2, (rows, k), generator=gen, dtype=torch.uint8) << 7
            return c.view(FP8).to(device)
        c = torch.randint(0, 256, (rows, k), generator=gen, dtype=torch.uint8)
        c[(c & 0x7f) == 0x7f] = 0x38
        # mostly ordinary values
        usual = (torch.randn(rows, k, generator=gen) * 90).clamp(-448, 448).to(FP8)
        pick = torch.rand(rows, k, generator=gen) < 0.1
        return torch.where(pick, c, usual.view(torch.uint8)).view(FP8).to(device)
    kb, nb = -(-k // 128), -(-n // 128)
    sa = torch.exp2(4 * torch.rand(m, kb, generator=gen) - 8).to(device)
    sw = torch.exp2(4 * torch.rand(nb, kb, generator=gen) - 8).to(device)
    return codes(m), sa, codes(n), sw


def _known_form(form):
    try:
        _capi.block_matmul_schedule(256, 256, 1024, form + 1)
    except ValueError:
        return False
    return True


def _product_ref(a, sa, w, sw, bias=None):
    k, n = a.shape[1], w.shape[0]
    a = a.double() * sa.double().repeat_interleave(128, 1)[:, :k]
    w = w.double() * sw.double().repeat_interleave(128, 1)[:, :k].repeat_interleave(128, 0)[:n]
    out, mag = a @ w.t(), a.abs() @ w.abs().t()
    if bias is not None:
        out, mag = out + bias.double(), mag + bias.double().abs()
    return out, mag


def _check_product(got, ref, mag, k, dtype, narrow=False):
    sums = (16 + 2 * -(-k // 128) + 2) * 2.0 ** -23 + (0.0 if narrow else 7 * 2.0 ** -13)
    bound = sums * (1 + HALF[dtype]) * mag + HALF[dtype] * ref.abs() + TINY[dtype]
    off = (got.double() - ref).abs() - bound
    assert got.dtype == dtype and not got.isnan().any()
    assert not (off > 0).any(), f"{float(off.max())} over the bound"


PRODUCT_SHAPES = [(1, 4096, 7168), (1, 1, 16), (1, 16, 128), (3, 17, 144), (16, 128, 256),
                  (17, 130, 272), (33, 576, 512), (48, 2112, 1552), (65, 100, 1024),
                  (128, 256, 2048), (200, 384, 640), (333, 2112, 1552), (257, 257, 272),
                  (512, 512, 128), (300, 1000, 16), (1000, 129, 3584)]


@pytest.mark.parametrize("m,n,k", PRODUCT_SHAPES)
def test_product(gpu, m, n, k):
    gen = torch.Generator().manual_seed(m + n + k)
    bias = torch.randn(n, generator=gen).to(gpu)
    for narrow in (True, False):
        a, sa, w, sw = _operands(gen, m, n, k, gpu, narrow)
        ref, mag = _product_ref(a, sa, w, sw)
        for dtype in (BF16, F16):
            _check_product(fgs.fp8_block_matmul(a, sa, w, sw, out_dtype=dtype), ref, mag, k,
                           dtype, narrow)
        for b in (bias, bias.to(BF16), bias.to(F16)):
            refb, magb = _product_ref(a, sa, w, sw, b)
            _check_product(fgs.fp8_block_matmul(a, sa, w, sw, bias=b), refb, magb, k, BF16,
                           narrow)


FORMS = [f for f in range(20) if _known_form(f)]
RAGGED = [(1, 1, 16), (70, 260, 144), (257, 257, 272), (130, 520, 1168), (300, 384, 640),
          (255, 1000, 128), (513, 130, 400), (64, 640, 2048)]


@pytest.mark.parametrize("m,n,k", RAGGED)
@pytest.mark.parametrize("form", FORMS)
def test_every_form_of_the_product(gpu, form, m, n, k):
    """Each kernel on sizes around its tiles' ends."""
    gen = torch.Generator().manual_seed(m * n + k)
    a, sa, w, sw = _operands(gen, m, n, k, gpu, narrow=True)
    bias = torch.randn(n, generator=gen).bfloat16().to(gpu)
    ref, mag = _product_ref(a, sa, w, sw)
    refb, magb = _product_ref(a, sa, w, sw, bias)
    got = fgs.fp8_block_matmul(a, sa, w, sw, out_dtype=F16, _flags=form + 1)
    _check_product(got, ref, mag, k, F16, narrow=True)
    got = fgs.fp8_block_matmul(a, sa.t().contiguous().t(), w, sw, bias=bias, _flags=form + 1)
    _check_product(got, refb, magb, k, BF16, narrow=True)


def _same(x, y):
    return torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("m", [5, 140, 600])
def test_product_of_strided_operands(gpu, m):
    """Scales with the rows adjacent, operands and output inside wider
    tensors, operands whose rows are not aligned, more dimensions."""
    gen = torch.Generator().manual_seed(m)
    n, k = 272, 384
    a, sa, w, sw = _operands(gen, m, n, k, gpu)
    ref = fgs.fp8_block_matmul(a, sa, w, sw)
    assert _same(fgs.fp8_block_matmul(a, sa.t().contiguous().t(), w, sw.t().contiguous().t()), ref)
    # the surroundings are NaN: nothing of them may be read into the result
    def inside(t, left, right):
        wide = torch.full((t.shape[0], t.shape[1] + left + right), 0x7f, dtype=torch.uint8,
                          device=gpu)
        wide[:, left:left + k] = t.view(torch.uint8)
        return wide.view(FP8)[:, left:left + k]
    assert _same(fgs.fp8_block_matmul(inside(a, 16, 32), sa, inside(w, 32, 0), sw), ref)
    assert _same(fgs.fp8_block_matmul(inside(a, 3, 2), sa, inside(w, 0, 9), sw), ref)
    for left in (4, 1):
        wide = torch.zeros(m, n + 8, dtype=BF16, device=gpu)
        out = wide[:, left:left + n]
        assert fgs.fp8_block_matmul(a, sa, w, sw, out=out) is out
        assert _same(out.contiguous(), ref)
        assert (wide[:, :left] == 0).all() and (wide[:, left + n:] == 0).all()
    cube = fgs.fp8_block_matmul(a.view(1, m, k), sa.view(1, m, -1), w, sw)
    assert cube.shape == (1, m, n) and _same(cube[0], ref)
    # a ragged k: what lies behind each row's end is not read
    ragged = fgs.fp8_block_matmul(inside(a, 0, 16)[:, :k - 48], sa, inside(w, 0, 16)[:, :k - 48],
                                  sw)
    cut = fgs.fp8_block_matmul(a[:, :k - 48].contiguous(), sa, w[:, :k - 48].contiguous(), sw)
    assert _same(ragged, cut) and not ragged.isnan().any()
    assert fgs.fp8_block_matmul(a[:0], sa[:0], w, sw).shape == (0, n)


def test_product_of_nans_stays_in_its_row_and_column(gpu):
    gen = torch.Generator().manual_seed(1)
    for m in (20, 300):
        a, sa, w, sw = _operands(gen, m, 272, 400, gpu)
        ref = fgs.fp8_block_matmul(a, sa, w, sw)
        a2, w2 = a.clone(), w.clone()
        a2.view(torch.uint8)[m - 1, 399] = 0x7f
        w2.view(torch.uint8)[271, 0] = 0xff
        out = fgs.fp8_block_matmul(a2, sa, w2, sw)
        assert out[m - 1].isnan().all() and out[:, 271].isnan().all()
        assert torch.equal(out[:m - 1, :271], ref[:m - 1, :271])


# ------------------------------------------------------------ run together ---
def _layer(gen, device):
    hidden, inter, experts, topk = 512, 256, 8, 2
    w = {}
    for name, shape in (("w13", (experts, 2 * inter, hidden)), ("w2", (experts, hidden, inter)),
                        ("s13", (1, 2 * inter, hidden)), ("s2", (1, hidden, inter))):
        q, s = quant.quantize_fp8_block((0.1 * torch.randn(shape, generator=gen)).to(device))
        w[name], w[name + "_scale"] = (q, s) if shape[0] > 1 else (q[0], s[0])
    w["norm"] = (1 + 0.1 * torch.randn(hidden, generator=gen)).bfloat16().to(device)
    w["router"] = torch.randn(hidden, experts, generator=gen).to(device) * 0.1
    return w, topk


def _run_layer(w, topk, x, residual):
    n = fgs.fused_rms_norm(x, w["norm"], 1e-6, residual, quant="fp8", return_norm=True)
    tw, ti = fgs.fused_topk(n.norm, n.norm.float() @ w["router"], topk)
    routed = fgs.fused_moe(n.norm, w["w13"], w["w2"], tw, ti, use_fp8_w8a8=True,
                           block_shape=[128, 128], w1_scale=w["w13_scale"],
                           w2_scale=w["w2_scale"])
    h = fgs.fp8_block_matmul(n.q, n.scales, w["s13"], w["s13_scale"])
    q, s = fgs.silu_and_mul_quant(h)
    shared = fgs.fp8_block_matmul(q, s, w["s2"], w["s2_scale"])
    return n, h, q, s, routed, shared, routed + shared


@pytest.mark.parametrize("m", [1, 19, 300])
def test_layer_of_routed_and_shared_experts(gpu, m):
    """The run a decoder layer makes: each step against the definition on its
    own inputs, and the shared expert against the routed experts' kernels given
    it as their only expert."""
    gen = torch.Generator().manual_seed(m)
    w, topk = _layer(gen, gpu)
    x, residual = (_rand(gen, (m, 512), BF16, gpu) for _ in range(2))
    n, h, q, s, routed, shared, out = _run_layer(w, topk, x, residual)
    href, nref = _norm_ref(x, w["norm"], 1e-6, residual, 0.0)
    _near(n.residual, href, HALF[BF16])
    _near(n.norm, nref, HALF[BF16], TINY[BF16])
    _check_codes(n.q, n.scales, nref, "fp8")
    ref, mag = _product_ref(n.q, n.scales, w["s13"], w["s13_scale"])
    _check_product(h, ref, mag, 512, BF16)
    _check_codes(q, s, _act_ref(h, False), "fp8")
    ref, mag = _product_ref(q, s, w["s2"], w["s2_scale"])
    _check_product(shared, ref, mag, 256, BF16)
    one = torch.zeros(m, 1, dtype=torch.int32, device=gpu)
    alone = fgs.fused_moe(n.norm, w["s13"][None], w["s2"][None], torch.ones(m, 1, device=gpu), one,
                          use_fp8_w8a8=True, block_shape=[128, 128],
                          w1_scale=w["s13_scale"][None], w2_scale=w["s2_scale"][None])
    # two e4m3 roundings (2^-4 each) of 512 and 256 independent terms
    # differ at most where the 16-bit norm does: far inside 2^-4 of the whole
    rel = (alone.double() - shared.double()).norm() / shared.double().norm()
    assert rel < 2.0 ** -4
    assert torch.equal(out, routed + shared)


@pytest.mark.parametrize("m", [1, 33, 300])
def test_layer_with_adjacent_scales(gpu, m):
    """The dense half with column-major scales: the bits of row-major ones."""
    gen = torch.Generator().manual_seed(m + 1)
    w, _ = _layer(gen, gpu)
    x, residual = (_rand(gen, (m, 512), BF16, gpu) for _ in range(2))
    out = []
    for column in (False, True):
        n = fgs.fused_rms_norm(x, w["norm"], 1e-6, residual, quant="fp8",
                               column_major_scales=column)
        assert n.scales.stride() == ((1, m) if column else (4, 1))
        h = fgs.fp8_block_matmul(n.q, n.scales, w["s13"], w["s13_scale"])
        q, s = fgs.silu_and_mul_quant(h, column_major_scales=column)
        out.append((n.q, n.scales, h, q, s, fgs.fp8_block_matmul(q, s, w["s2"], w["s2_scale"])))
    for a, b in zip(*out):
        assert _same(a.contiguous(), b.contiguous())


def test_layer_replayed_from_a_graph(gpu):
    """Captured once, replayed several times on new inputs with eager calls
    between; every replay gives the eager bits."""
    gen = torch.Generator().manual_seed(77)
    w, topk = _layer(gen, gpu)
    for m in (4, 200):
        x, residual = (_rand(gen, (m, 512), BF16, gpu) for _ in range(2))
        _run_layer(w, topk, x, residual)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = _run_layer(w, topk, x, residual)[-1]
        for i in range(4):
            fresh = [_rand(gen, (m, 512), BF16, gpu) for _ in range(2)]
            x.copy_(fresh[0])
            residual.copy_(fresh[1])
            eager = _run_layer(w, topk, *fresh)[-1]
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, eager), (m, i)


def test_two_streams_at_once(gpu):
    """Calls on streams of their own."""
    gen = torch.Generator().manual_seed(3)
    jobs = []
    for m, n, k in ((256, 512, 2048), (130, 1024, 4096)):
        args = _operands(gen, m, n, k, gpu)
        jobs.append((args, fgs.fp8_block_matmul(*args), torch.cuda.Stream()))
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for args, ref, stream in jobs:
            with torch.cuda.stream(stream):
                got.append((fgs.fp8_block_matmul(*args), ref))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in got)


# ----------------------------------------------------- calls less ordinary ---
def test_one_tensor_as_both_inputs(gpu):
    """The residual is the input itself, replaced in place or not; rows that
    are one row repeated; weights that lie apart."""
    gen = torch.Generator().manual_seed(8)
    for rows, cols in ((3, 200), (1030, 512), (2, 40000)):
        x = _rand(gen, (rows, cols), BF16, gpu)
        w = _rand(gen, (cols, 2), BF16, gpu, loud=False)[:, 1]
        h, n = _norm_ref(x, w, 1e-6, x, 0.0)
        plain = fgs.fused_rms_norm(x, w, residual=x, quant="int8", return_norm=True)
        _near(plain.residual, h, HALF[BF16])
        _near(plain.norm, n, HALF[BF16], TINY[BF16])
        row = x[:1].expand(rows, cols)
        flat = fgs.fused_rms_norm(row, w, residual=x)
        again = fgs.fused_rms_norm(row.contiguous(), w, residual=x)
        assert _same(flat.norm, again.norm) and _same(flat.residual, again.residual)
        version = x._version
        o = fgs.fused_rms_norm(x, w, residual=x, quant="int8", return_norm=True, inplace=True)
        assert o.residual is x and x._version > version
        assert all(_same(a, b) for a, b in zip(o, plain))


def test_expanded_operands_of_the_product(gpu):
    gen = torch.Generator().manual_seed(12)
    for m in (7, 300):
        a, sa, w, sw = _operands(gen, m, 272, 400, gpu)
        bias = torch.randn(1, generator=gen).to(gpu).expand(272)
        got = fgs.fp8_block_matmul(a[:1].expand(m, 400), sa[:1].expand(m, 4), w, sw, bias=bias)
        ref = fgs.fp8_block_matmul(a[:1].repeat(m, 1), sa[:1].repeat(m, 1), w, sw,
                                   bias=bias.contiguous())
        assert _same(got, ref)
        got = fgs.fp8_block_matmul(a, sa[:, :1].expand(m, 4), w, sw[:1, :1].expand(3, 4))
        ref = fgs.fp8_block_matmul(a, sa[:, :1].repeat(1, 4), w, sw[:1, :1].repeat(3, 4))
        assert _same(got, ref)


def test_no_rows(gpu):
    x = torch.zeros(2, 0, 512, dtype=BF16, device=gpu)
    w = torch.ones(512, device=gpu)
    for kind in ("fp8", "int8"):
        o = fgs.fused_rms_norm(x, w, quant=kind, residual=x, inplace=True,
                               column_major_scales=True)
        assert o.residual is x and o.q.shape == x.shape
        assert o.scales.shape == ((2, 0, 4) if kind == "fp8" else (2, 0))
        q, s = fgs.silu_and_mul_quant(x, kind, column_major_scales=True)
        assert q.shape == (2, 0, 256) and s.shape == ((2, 0, 2) if kind == "fp8" else (2, 0))
    q, s = fgs.silu_and_mul_quant(x)
    weights = torch.zeros(48, 256, device=gpu).to(FP8)
    out = torch.empty(2, 0, 48, dtype=F16, device=gpu)
    assert fgs.fp8_block_matmul(q, s, weights, torch.ones(1, 2, device=gpu), out=out) is out


def test_refusals_of_gpu_tensors(gpu):
    gen = torch.Generator().manual_seed(4)
    x = _rand(gen, (4, 256), F32, gpu)
    w = torch.ones(256, device=gpu)
    a, sa, b, sb = _operands(gen, 4, 272, 256, gpu)
    leaf = x.clone().requires_grad_()
    for call in (lambda: fgs.fused_rms_norm(leaf, w), lambda: fgs.silu_and_mul_quant(leaf),
                 lambda: fgs.fused_rms_norm(x, w.clone().requires_grad_()),
                 lambda: fgs.fused_rms_norm(x, w, residual=leaf, inplace=True),
                 lambda: fgs.fp8_block_matmul(a, sa, b, sb, bias=torch.ones(
                     272, device=gpu, requires_grad=True))):
        with pytest.raises(RuntimeError, match="no backward"):
            call()
        with torch.no_grad():
            call()
    with torch.inference_mode():
        y = x.clone()
        assert _same(fgs.fused_rms_norm(y, w, residual=y, inplace=True).residual, x + x)
    negated = torch.complex(x, x).conj().imag
    assert negated.is_neg()
    with pytest.raises(NotImplementedError, match="negated"):
        fgs.fused_rms_norm(negated, w)
    with pytest.raises(RuntimeError, match="weight is on cpu"):
        fgs.fused_rms_norm(x, w.cpu())
    with pytest.raises(RuntimeError, match="out is on cpu"):
        fgs.fp8_block_matmul(a, sa, b, sb, out=torch.empty(4, 272, dtype=BF16))
    for text, kw in (("x's type", dict(weight=w.to(BF16))), ("weight must be", dict(weight=w[:8])),
                     ("x's shape", dict(residual=x[:2])), ("needs a residual", dict(inplace=True)),
                     ("no output", dict(return_norm=False))):
        with pytest.raises(AssertionError, match=text):
            fgs.fused_rms_norm(**{"x": x, "weight": w, **kw})
    with pytest.raises(ValueError, match="evenly spaced"):
        fgs.fused_rms_norm(x, w, residual=x[:1].expand(4, 256), inplace=True)
    with pytest.raises(ValueError, match="evenly spaced"):
        fgs.fused_rms_norm(x, w, residual=x.t().contiguous().t(), inplace=True)
    with pytest.raises(AssertionError, match="gate half"):
        fgs.silu_and_mul_quant(x[:, :255])
    with pytest.raises(NotImplementedError, match="65536"):
        fgs.fused_rms_norm(torch.zeros(1, 65544, device=gpu), torch.ones(65544, device=gpu))
    for text, args, kw in (
            ("float8", (a.float(), sa, b, sb), {}), ("must be", (a, sa, b[:, :128], sb), {}),
            ("a_scale must", (a, sa[:, :1], b, sb), {}), ("w_scale must", (a, sa, b, sb[:2]), {}),
            ("float32", (a, sa.double(), b, sb), {}), ("bias must", (a, sa, b, sb),
                                                       dict(bias=torch.ones(271, device=gpu))),
            ("bfloat16 or float16", (a, sa, b, sb), dict(out_dtype=F32)),
            ("out must", (a, sa, b, sb), dict(out=torch.empty(4, 271, dtype=BF16, device=gpu)))):
        with pytest.raises(AssertionError, match=text):
            fgs.fp8_block_matmul(*args, **kw)
    for out in (torch.empty(272, 4, dtype=BF16, device=gpu).t(),
                torch.empty(1, 272, dtype=BF16, device=gpu).expand(4, 272)):
        with pytest.raises(ValueError, match="out must be adjacent|ldo"):
            fgs.fp8_block_matmul(a, sa, b, sb, out=out)
    with pytest.raises(ValueError, match="k >= 1"):
        fgs.fp8_block_matmul(a[:, :0], sa[:, :0], b[:, :0], sb[:, :0])
    with pytest.raises(NotImplementedError, match="multiple of 16"):
        fgs.fp8_block_matmul(a[:, :136], sa, b[:, :136], sb)


def test_threads_call_at_once(gpu):
    """Two Python threads (the calls leave the interpreter's lock), each on a
    stream of its own, get what one thread gets."""
    gen = torch.Generator().manual_seed(6)
    w, topk = _layer(gen, gpu)
    jobs = []
    for m in (1, 33):
        x, residual = (_rand(gen, (m, 512), BF16, gpu) for _ in range(2))
        jobs.append((x, residual, _run_layer(w, topk, x, residual)[-2]))
    torch.cuda.synchronize()
    wrong = []

    def work(x, residual, ref):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                n = fgs.fused_rms_norm(x, w["norm"], 1e-6, residual, quant="fp8")
                q, s = fgs.silu_and_mul_quant(
                    fgs.fp8_block_matmul(n.q, n.scales, w["s13"], w["s13_scale"]))
                got = fgs.fp8_block_matmul(q, s, w["s2"], w["s2_scale"])
                torch.cuda.current_stream().synchronize()
                if not torch.equal(got, ref):
                    wrong.append(x.shape)

    threads = [threading.Thread(target=work, args=job) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


# ------------------------------------------------------ offsets past 2^31 ---
def _picked(rows, cols):
    """Rows on both sides of element 2^31, and the ends."""
    edge = 2 ** 31 // cols
    assert rows > edge + 1
    return torch.tensor([0, edge - 1, edge, edge + 1, rows - 1])


def test_norm_past_31_bits(gpu):
    rows, cols = 65540, 32768
    gen = torch.Generator(device=gpu).manual_seed(1)
    x = torch.randn(rows, cols, device=gpu, dtype=BF16, generator=gen)
    w = torch.randn(cols, device=gpu, dtype=BF16, generator=gen)
    at = _picked(rows, cols).to(gpu)
    h, n = _norm_ref(x[at], w, 1e-6, x[at], 0.0)
    for kind in ("fp8", "int8"):
        o = fgs.fused_rms_norm(x, w, residual=x, quant=kind, return_norm=True)
        _near(o.residual[at], h, HALF[BF16])
        _near(o.norm[at], n, HALF[BF16], TINY[BF16])
        _check_codes(o.q.view(torch.uint8)[at].view(o.q.dtype), o.scales[at], n, kind)


def test_activation_past_31_bits(gpu):
    rows, n = 65540, 32768
    gen = torch.Generator(device=gpu).manual_seed(2)
    x = torch.randn(rows, 2 * n, device=gpu, dtype=BF16, generator=gen)
    at = _picked(rows, n).to(gpu)
    ref = _act_ref(x[at], False)
    for kind in ("fp8", "int8"):
        q, s = fgs.silu_and_mul_quant(x, kind)
        _check_codes(q.view(torch.uint8)[at].view(q.dtype), s[at], ref, kind)


@pytest.mark.parametrize("m,n,k,what", [(262149, 32, 8192, "a"), (40000, 65536, 16, "out"),
                                        (2, 65540, 32768, "w"), (300, 65540, 32768, "w")])
def test_product_past_31_bits(gpu, m, n, k, what):
    gen = torch.Generator(device=gpu).manual_seed(m)

    def codes(rows):
        c = torch.randint(0x38, 0x58, (rows, k), generator=gen, dtype=torch.uint8, device=gpu)
        c |= torch.randint(0, 2, (rows, k), generator=gen, dtype=torch.uint8, device=gpu) << 7
        return c.view(FP8)
    a, w = codes(m), codes(n)
    sa, sw = (torch.exp2(4 * torch.rand(r, -(-k // 128), generator=gen, device=gpu) - 8)
              for r in (m, -(-n // 128)))
    out = fgs.fp8_block_matmul(a, sa, w, sw)
    rows = _picked(m, k if what == "a" else n).to(gpu) if what != "w" else torch.arange(
        m, device=gpu)[-64:]
    cols = _picked(n, k).to(gpu) if what == "w" else torch.arange(n, device=gpu)[-64:]
    pick_w, pick_sw = w.view(torch.uint8)[cols].view(FP8), sw[cols // 128]
    pick_a, pick_sa = a.view(torch.uint8)[rows].view(FP8), sa[rows]
    x = pick_a.double() * pick_sa.double().repeat_interleave(128, 1)[:, :k]
    y = pick_w.double() * pick_sw.double().repeat_interleave(128, 1)[:, :k]
    _check_product(out[rows][:, cols], x @ y.t(), x.abs() @ y.abs().t(), k, BF16, narrow=True)
