"""Refusals and schedules of the dense operators: no GPU is touched (the
library checks its arguments before any launch)."""

import ctypes

import pytest
import torch

from flaggems_sglang import _capi, fp8_block_matmul, fused_rms_norm, quant, silu_and_mul_quant

P = 0x1000  # an address no call reads


def _norm(**kw):
    a = dict(x=P, x_stride=256, residual=None, r_stride=0, weight=P, dtype=0, wdtype=0, eps=1e-6,
             offset=0.0, rows=4, cols=256, norm=P, res_out=None, ro_stride=0, quant=0, q=None,
             scales=None, s_row=2, s_col=1)
    a.update(kw)
    rc = _capi.load().fgs_moe_rms_norm(*a.values(), None)
    return rc, _capi.last_error()


@pytest.mark.parametrize("kw,rc,text", [
    (dict(rows=-1), -1, "rows >= 0"),
    (dict(cols=0), -1, "cols >= 1"),
    (dict(cols=65537), -2, "more than 65536"),
    (dict(rows=1 << 31), -2, "too many rows"),
    (dict(dtype=3), -1, "unknown element type"),
    (dict(dtype=0, wdtype=1), -2, "weight must be"),
    (dict(quant=3, q=P, scales=P), -1, "unknown quantisation"),
    (dict(quant=1, q=P), -1, "null pointer"),
    (dict(quant=1, scales=P), -1, "null pointer"),
    (dict(q=P, scales=P), -1, "need a quantisation"),
    (dict(x=None), -1, "null pointer"),
    (dict(weight=None), -1, "null pointer"),
    (dict(residual=P, r_stride=256), -1, "residual_out is needed"),
    (dict(residual=P, r_stride=256, res_out=P, ro_stride=255), -1, "row strides"),
    (dict(x_stride=-1), -1, "row strides"),
    (dict(norm=None), -1, "no output"),
    (dict(x=P + 1), -1, "aligned"),
    (dict(dtype=2, wdtype=2, x=P + 2), -1, "aligned"),
    (dict(weight=P + 2, wdtype=2), -1, "aligned"),
    (dict(quant=2, q=P, scales=P + 2), -1, "aligned"),
    (dict(rows=0, x=None, norm=None), 0, ""),
])
def test_norm_refusals(kw, rc, text):
    got, msg = _norm(**kw)
    assert got == rc
    assert rc == 0 or text in msg


def _act(**kw):
    a = dict(x=P, x_stride=512, dtype=0, rows=4, n=256, gelu=0, quant=1, q=P, scales=P, s_row=2,
             s_col=1)
    a.update(kw)
    rc = _capi.load().fgs_moe_silu_and_mul_quant(*a.values(), None)
    return rc, _capi.last_error()


@pytest.mark.parametrize("kw,rc,text", [
    (dict(rows=-1), -1, "rows >= 0"),
    (dict(n=0), -1, "cols >= 1"),
    (dict(n=65537), -2, "more than 65536"),
    (dict(dtype=9), -1, "unknown element type"),
    (dict(quant=0), -1, "unknown quantisation"),
    (dict(q=None), -1, "null pointer"),
    (dict(x=None), -1, "null pointer"),
    (dict(x_stride=-4), -1, "row strides"),
    (dict(x=P + 1), -1, "aligned"),
    (dict(rows=0, x=None, q=None, scales=None), 0, ""),
])
def test_activation_refusals(kw, rc, text):
    got, msg = _act(**kw)
    assert got == rc
    assert rc == 0 or text in msg


def _product(**kw):
    a = dict(a=P, lda=256, a_scale=P, as_row=2, as_col=1, w=P, ldw=256, w_scale=P, bias=None,
             bias_dtype=0, m=4, n=512, k=256, out_dtype=0, flags=0, out=P, ldo=512)
    a.update(kw)
    rc = _capi.load().fgs_moe_fp8_block_matmul(*a.values(), None)
    return rc, _capi.last_error()


@pytest.mark.parametrize("kw,rc,text", [
    (dict(m=-1), -1, "m >= 0"),
    (dict(n=0), -1, "n >= 1"),
    (dict(k=0), -1, "k >= 1"),
    (dict(k=200), -2, "multiple of 16"),
    (dict(m=1 << 23), -2, "too large"),
    (dict(n=1 << 23), -2, "too large"),
    (dict(k=1 << 25), -2, "too large"),
    (dict(lda=1 << 23), -2, "stride too large"),
    (dict(ldw=1 << 23), -2, "stride too large"),
    (dict(as_row=1 << 21), -2, "stride too large"),
    (dict(as_col=-1), -2, "stride too large"),
    (dict(flags=1 << 20), -1, "unknown flags"),
    (dict(flags=-1), -1, "unknown flags"),
    (dict(out_dtype=5), -1, "unknown element type"),
    (dict(bias=P, bias_dtype=-1), -1, "unknown element type"),
    (dict(a=None), -1, "null pointer"),
    (dict(w_scale=None), -1, "null pointer"),
    (dict(out=None), -1, "null pointer"),
    (dict(lda=250), -2, "16-byte aligned"),
    (dict(lda=-256), -2, "16-byte aligned"),
    (dict(ldw=264), -2, "16-byte aligned"),
    (dict(a=P + 8), -2, "16-byte aligned"),
    (dict(w=P + 8), -2, "16-byte aligned"),
    (dict(ldo=511), -1, "ldo"),
    (dict(out=P + 1), -1, "aligned to their elements"),
    (dict(out_dtype=2), -2, "bf16 or fp16"),
    (dict(m=0, a=None, out=None), 0, ""),
])
def test_product_refusals(kw, rc, text):
    got, msg = _product(**kw)
    assert got == rc
    assert rc == 0 or text in msg


def test_schedule_text():
    lib = _capi.load()
    assert lib.fgs_moe_fp8_block_matmul_schedule(1, 1, 16, 0, None, 0) == _capi.FGS_EINVAL
    buf = ctypes.create_string_buffer(5)
    assert lib.fgs_moe_fp8_block_matmul_schedule(1, 4096, 7168, 0, buf, 5) == 0
    assert buf.value == b"stre"
    with pytest.raises(NotImplementedError):
        _capi.block_matmul_schedule(1, 1, 8)


@pytest.mark.parametrize("m,n,k,schedule", [
    (0, 4096, 7168, "none"), (1, 16384, 7168, "stream 16x16"),
    (16, 4096, 7168, "stream 16x16"), (32, 4096, 7168, "stream 32x16"),
    (64, 4096, 7168, "stream 32x32"), (128, 4096, 7168, "stream 64x32"),
    (256, 4096, 7168, "stream 64x64"), (512, 4096, 7168, "tiled 64x128"),
    (1024, 4096, 7168, "tiled 128x128 deep"), (2048, 4096, 7168, "tiled 128x256"),
    (3600, 1828, 384, "tiled 128x128"), (4096, 4096, 7168, "tiled 256x256"),
    (8192, 14336, 7168, "tiled 256x256"),
])
def test_schedules(m, n, k, schedule):
    """The tile of a product by the sizes' estimate (the shapes the estimate
    was measured on)."""
    assert _capi.block_matmul_schedule(m, n, k) == schedule


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 256)
    q = torch.zeros(2, 256, dtype=torch.float8_e4m3fn)
    s = torch.ones(2, 2)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        fused_rms_norm(x, x[0])
    with pytest.raises(RuntimeError, match="GPU tensor"):
        silu_and_mul_quant(x)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        fp8_block_matmul(q, s, q, s[:1])


def test_registered():
    import flaggems_sglang

    for name in ("fused_rms_norm", "silu_and_mul_quant", "fp8_block_matmul"):
        assert flaggems_sglang.get_op(name) is getattr(flaggems_sglang, name)


def test_grids_the_runtime_cannot_count():
    """A grid's threads are counted in 32 bits."""
    rows = (1 << 31) - 1
    for rc, msg in (_norm(rows=rows, cols=4096), _norm(rows=rows), _act(rows=rows),
                    _product(m=1 << 22, n=1 << 22, ldo=1 << 22),
                    _product(m=1 << 22, n=1 << 14, ldo=1 << 14, flags=1)):
        assert rc == -2 and "for a grid" in msg


def test_host_module_arguments():
    host = _capi.host()
    with pytest.raises(TypeError, match="9 arguments expected, got 1"):
        host.rms_norm(1)
    with pytest.raises(TypeError, match="a must be a tensor"):
        fp8_block_matmul(None, None, None, None)
    with pytest.raises(TypeError, match="residual must be a tensor"):
        fused_rms_norm(torch.zeros(1, 8), torch.zeros(8), 1e-6, 3)
    for bad in ("fp4", 1):
        with pytest.raises(ValueError, match="quantisation"):
            fused_rms_norm(torch.zeros(1, 8), torch.zeros(8), quant=bad)
        with pytest.raises(ValueError, match="quantisation"):
            silu_and_mul_quant(torch.zeros(1, 8), bad)
    with pytest.raises(ValueError, match="quantisation"):
        silu_and_mul_quant(torch.zeros(1, 8), None)
    with pytest.raises(ValueError, match="activation"):
        silu_and_mul_quant(torch.zeros(1, 8), activation="relu")


@pytest.mark.parametrize("r,c", [(128, 256), (1, 16), (300, 208), (129, 128)])
def test_dense_weights_in_blocks(r, c):
    """A matrix of any size: each block's scale is its largest magnitude over
    448, and its codes are its values over that (as an expert's weights)."""
    w = torch.randn(r, c, generator=torch.Generator().manual_seed(r))
    q, s = quant.quantize_fp8_block(w)
    assert q.shape == (r, c) and q.is_contiguous() and s.shape == (-(-r // 128), -(-c // 128))
    for i in range(s.shape[0]):
        for j in range(s.shape[1]):
            b = w[128 * i:128 * i + 128, 128 * j:128 * j + 128]
            scale = b.abs().max() / 448
            assert s[i, j] == scale
            got = q[128 * i:128 * i + 128, 128 * j:128 * j + 128]
            assert torch.equal(got.float(), (b / scale).to(torch.float8_e4m3fn).float())
    if r % 128 == 0 and c % 128 == 0:
        q3, s3 = quant.quantize_fp8_block(w[None])
        assert torch.equal(q3[0].float(), q.float()) and torch.equal(s3[0], s)
