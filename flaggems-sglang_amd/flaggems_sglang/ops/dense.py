"""Dense operators around the routed experts for MI355X (gfx950).

A decoder layer whose weights are e4m3 with a scale per 128x128 block adds
the residual and normalises it, feeds the 16-bit norm to the router and the
routed experts (:mod:`flaggems_sglang.ops.fused_moe`) and an 8-bit copy of it
to dense products -- the shared expert's, the projections'::

    n = fused_rms_norm(x, weight, eps, residual, quant="fp8", return_norm=True)
    routed = fused_moe(n.norm, w13, w2, *fused_topk(...), use_fp8_w8a8=True, ...)
    h = fp8_block_matmul(n.q, n.scales, shared_w13, shared_w13_scale)
    q, s = silu_and_mul_quant(h)
    out = routed + fp8_block_matmul(q, s, shared_w2, shared_w2_scale)

The host side validates tensors, allocates outputs and workspaces with the
torch caching allocator and hands pointers and the current HIP stream to
``libfgs_moe.so`` (include/fgs_moe.h). There is no CPU path. None of these
has a backward pass: outputs are cut from the autograd graph, and an input
that requires a gradient is refused while gradients are recorded.

The reference has no counterparts (its layer takes its input normalised, and
src/flaggems_sglang/ops/fused_moe.py:170-185 rejects every 8-bit mode).
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from flaggems_sglang import _capi
from flaggems_sglang.ops.fused_moe import _require_gpu, _stream_ptr

_DTYPES = {torch.bfloat16: _capi.DTYPE_BF16, torch.float16: _capi.DTYPE_FP16,
           torch.float32: _capi.DTYPE_FP32}
_QUANTS = {None: _capi.QUANT_NONE, "fp8": _capi.QUANT_FP8_GROUP,
           "int8": _capi.QUANT_INT8_TOKEN}
_CODES = {_capi.QUANT_FP8_GROUP: torch.float8_e4m3fn, _capi.QUANT_INT8_TOKEN: torch.int8}
_GROUP = 128  # columns of an e4m3 scale
# Largest row strides of the product's operands and of its activation scales
_MAX_STRIDE, _MAX_SCALE_STRIDE = 1 << 22, 1 << 20


class RMSNormOutput(NamedTuple):
    """What :func:`fused_rms_norm` returns; what a call does not make is None."""

    norm: Optional[torch.Tensor]
    residual: Optional[torch.Tensor]
    q: Optional[torch.Tensor]
    scales: Optional[torch.Tensor]


# torch's current device index: the accessor behind current_device(), or that
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _check_inputs(names: str, first: torch.Tensor, *others: Optional[torch.Tensor]) -> int:
    """Every tensor given is on one GPU and needs no gradient; that GPU's
    index. ``names``: the tensors' names, for the messages."""
    if not first.is_cuda:
        _require_gpu(names.split()[0], first)
    index = first.get_device()
    for i, t in enumerate(others):
        if t is not None and t.get_device() != index:
            raise RuntimeError(f"{names.split()[i + 1]} is on {t.device}, not on {first.device}")
    if torch.is_grad_enabled():
        for i, t in enumerate((first,) + others):
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{names.split()[i]} requires a gradient: this operator has "
                                   "no backward pass (call it under torch.no_grad())")
    return index


def _call(index: int, what: str, fn, *args) -> None:
    """Runs a library entry on GPU ``index`` (whichever one is current)."""
    if index == _current_device():
        rc = fn(*args)
    else:
        with torch.cuda.device(index):
            rc = fn(*args)
    if rc:
        _capi.check(rc, what)


def _written(t: torch.Tensor) -> None:
    """Tells autograd that the library has written a caller's tensor."""
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)


def _rows(x: torch.Tensor, cols: int):
    """``x`` as rows of its last dimension: (tensor whose storage they are in,
    row stride in elements). Rows that lie evenly spaced, as those of a slice
    of a wider tensor, are taken where they are."""
    if x.is_contiguous():
        return x, cols
    if x.ndim == 2 and (x.stride(1) == 1 or cols == 1):
        return x, x.stride(0)
    return x.contiguous(), cols


def _like(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """An uninitialised contiguous tensor of x's shape."""
    if x.is_contiguous():
        return torch.empty_like(x, dtype=dtype)
    return torch.empty(x.shape, dtype=dtype, device=x.device)


def _scales_like(x: torch.Tensor, rows: int, cols: int, mode: int, column_major: bool):
    """``(scales, stride over rows, over groups)`` of the rows of x."""
    lead = x.shape[:-1]
    if mode == _capi.QUANT_INT8_TOKEN:
        return x.new_empty(lead, dtype=torch.float32), 1, 0
    groups = (cols + _GROUP - 1) // _GROUP
    if not column_major:
        return x.new_empty(lead + (groups,), dtype=torch.float32), groups, 1
    scales = x.new_empty((groups, rows), dtype=torch.float32).t()
    return scales if x.ndim == 2 else scales.view(lead + (groups,)), 1, rows


def fused_rms_norm(
    x: torch.Tensor,
    weight: torch.Tensor,
    eps: float = 1e-6,
    residual: Optional[torch.Tensor] = None,
    *,
    weight_offset: float = 0.0,
    quant: Optional[str] = None,
    return_norm: Optional[bool] = None,
    column_major_scales: bool = False,
    inplace: bool = False,
) -> RMSNormOutput:
    """Root-mean-square norm of the rows of ``x [..., cols]``, with the
    residual's addition before it and an output in 8 bits after it::

        h = x + residual                                (residual output)
        n = h / sqrt(mean(h^2) + eps) * (weight + weight_offset)

    in fp32; each output is rounded once. ``x`` and ``residual`` (of x's
    shape) bf16, fp16 or fp32, ``weight [cols]`` of x's type or fp32;
    ``weight_offset=1`` for weights stored about zero. ``cols`` up to 65536;
    multiples of 8 with 16-byte aligned rows run fastest.

    ``quant="fp8"``: ``q`` e4m3fn with ``scales [..., ceil(cols / 128)]`` per
    128 columns, ``"int8"``: ``q`` int8 with ``scales [...]`` per row (the
    codes of ``per_token_group_quant_fp8`` / ``per_token_quant_int8``, here of
    the unrounded ``n``). ``column_major_scales`` lays e4m3 scales out with
    the rows adjacent. ``return_norm``: whether ``n`` comes back in x's type
    (default: where nothing is quantised). ``inplace``: the sum replaces
    ``residual``'s values and ``residual`` is the residual output.

    A NaN in a row makes its outputs NaN (int8 codes 0, scale NaN). Returns
    ``RMSNormOutput(norm, residual, q, scales)``.
    """
    index = _check_inputs("x weight residual", x, weight, residual)
    mode = _QUANTS.get(quant)
    if mode is None:
        raise ValueError(f"Unsupported quantisation: {quant}")
    dtype = x.dtype
    assert dtype in _DTYPES, "x must be bfloat16, float16 or float32"
    assert x.ndim >= 1 and x.shape[-1] > 0, "x must have columns"
    cols = x.shape[-1]
    assert weight.shape == (cols,), "weight must be [cols]"
    assert weight.dtype == dtype or weight.dtype == torch.float32, (
        "weight must be of x's type or float32")
    if return_norm is None:
        return_norm = quant is None
    assert return_norm or mode or residual is not None, "no output was asked for"
    rows = x.numel() // cols
    xr, x_stride = _rows(x, cols)
    r_ptr = out_ptr = None
    r_stride = out_stride = 0
    res_out = None
    if residual is not None:
        assert residual.shape == x.shape and residual.dtype == dtype, (
            "residual must be of x's shape and type")
        rr, r_stride = _rows(residual, cols)
        r_ptr = rr.data_ptr()
        if inplace:
            if rr is not residual or (rows > 1 and r_stride < cols):
                raise ValueError("fused_rms_norm: an inplace residual must have evenly spaced "
                                 "rows that do not overlap")
            res_out, out_stride = residual, r_stride
        else:
            res_out, out_stride = _like(x, dtype), cols
        out_ptr = res_out.data_ptr()
    else:
        assert not inplace, "inplace needs a residual"
    norm = q = scales = norm_ptr = q_ptr = scales_ptr = None
    s_row = s_col = 0
    if return_norm:
        norm = _like(x, dtype)
        norm_ptr = norm.data_ptr()
    if mode:
        q = _like(x, _CODES[mode])
        scales, s_row, s_col = _scales_like(x, rows, cols, mode, column_major_scales)
        q_ptr = q.data_ptr()
        scales_ptr = scales.data_ptr()
    weight = weight.contiguous()
    _call(index, "fused_rms_norm", _capi.load().fgs_moe_rms_norm,
          xr.data_ptr(), x_stride, r_ptr, r_stride, weight.data_ptr(), _DTYPES[dtype],
          _DTYPES[weight.dtype], eps, weight_offset, rows, cols, norm_ptr, out_ptr, out_stride,
          mode, q_ptr, scales_ptr, s_row, s_col, _stream_ptr(x))
    if inplace:
        _written(residual)
    return RMSNormOutput(norm, res_out, q, scales)


def silu_and_mul_quant(
    x: torch.Tensor,
    quant: str = "fp8",
    *,
    activation: str = "silu",
    column_major_scales: bool = False,
):
    """``act(gate) * up`` over ``x = [gate | up]`` (``[..., 2n]``, bf16, fp16
    or fp32) in 8 bits: ``silu_and_mul`` and a quantiser in one pass, the
    codes taken from the unrounded fp32 product.

    ``activation``: "silu", or "gelu" (exact, erf). ``quant`` and
    ``column_major_scales`` as for :func:`fused_rms_norm`; ``n`` up to 65536.
    Returns ``(q [..., n], scales)``.
    """
    index = _check_inputs("x", x)
    if activation not in ("silu", "gelu"):
        raise ValueError(f"Unsupported activation: {activation}")
    mode = _QUANTS.get(quant)
    if not mode:
        raise ValueError(f"Unsupported quantisation: {quant}")
    assert x.dtype in _DTYPES, "x must be bfloat16, float16 or float32"
    assert x.ndim >= 1 and x.shape[-1] % 2 == 0 and x.shape[-1] > 0, (
        "x must hold a gate half and an up half")
    n = x.shape[-1] // 2
    rows = x.numel() // (2 * n)
    xr, x_stride = _rows(x, 2 * n)
    q = x.new_empty(x.shape[:-1] + (n,), dtype=_CODES[mode])
    scales, s_row, s_col = _scales_like(x, rows, n, mode, column_major_scales)
    _call(index, "silu_and_mul_quant", _capi.load().fgs_moe_silu_and_mul_quant,
          xr.data_ptr(), x_stride, _DTYPES[x.dtype], rows, n, activation == "gelu", mode,
          q.data_ptr(), scales.data_ptr(), s_row, s_col, _stream_ptr(x))
    return q, scales


def _byte_rows(t: torch.Tensor, cols: int):
    """An e4m3 matrix with adjacent columns and 16-byte aligned rows, and its
    row stride: where it is, or copied."""
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous() and cols % 16 == 0:
            return t, cols
        if t.stride(1) == 1 and (t.shape[0] <= 1 or (t.stride(0) % 16 == 0
                                                      and t.stride(0) <= _MAX_STRIDE)):
            return t, t.stride(0)
    return t.clone(memory_format=torch.contiguous_format), cols


def fp8_block_matmul(
    a: torch.Tensor,
    a_scale: torch.Tensor,
    w: torch.Tensor,
    w_scale: torch.Tensor,
    *,
    bias: Optional[torch.Tensor] = None,
    out_dtype: torch.dtype = torch.bfloat16,
    out: Optional[torch.Tensor] = None,
    _flags: int = 0,
) -> torch.Tensor:
    """``a @ w.T`` of e4m3 matrices with a scale for each block of 128::

        out[i, j] = sum_kb a_scale[i, kb] * w_scale[j // 128, kb]
                    * sum_{l in kb} a[i, l] * w[j, l]   (+ bias[j])

    ``a [..., k]`` with ``a_scale [..., ceil(k / 128)]`` (what
    ``per_token_group_quant_fp8``, :func:`fused_rms_norm` and
    :func:`silu_and_mul_quant` return, row- or column-major), ``w [n, k]``
    with ``w_scale [ceil(n / 128), ceil(k / 128)]``
    (``quant.quantize_fp8_block``). ``k`` is a multiple of 16, ``n`` and the
    number of rows are any. Sums are fp32 (of groups of eight products that the
    matrix instruction aligns to the largest and cuts 13 bits below it),
    ``bias [n]`` (fp32, bf16 or fp16) is added to them, and the result is
    rounded once to ``out_dtype`` (bf16 or fp16). ``out``: a tensor of that type and shape to write, whose
    rows may lie apart (2-D).
    """
    index = _check_inputs("a a_scale w w_scale bias out", a, a_scale, w, w_scale, bias, out)
    assert a.dtype == torch.float8_e4m3fn and w.dtype == torch.float8_e4m3fn, (
        "a and w must be float8_e4m3fn")
    assert w.ndim == 2 and a.ndim >= 1 and a.shape[-1] == w.shape[1], (
        "a must be [..., k] and w [n, k]")
    n, k = w.shape
    kb = (k + _GROUP - 1) // _GROUP
    lead = a.shape[:-1]
    assert a_scale.shape == lead + (kb,), "a_scale must be [..., ceil(k / 128)]"
    assert w_scale.shape == ((n + _GROUP - 1) // _GROUP, kb), (
        "w_scale must be [ceil(n / 128), ceil(k / 128)]")
    assert a_scale.dtype == torch.float32 and w_scale.dtype == torch.float32, (
        "scales must be float32")
    given = out is not None
    if given:
        out_dtype = out.dtype
        assert out.shape == lead + (n,), "out must be [..., n]"
        if out.stride(1) != 1 and n > 1 if out.ndim == 2 else not out.is_contiguous():
            raise ValueError("fp8_block_matmul: the columns of out must be adjacent")
    assert out_dtype == torch.bfloat16 or out_dtype == torch.float16, (
        "the output must be bfloat16 or float16")
    bias_ptr, bias_type = None, 0
    if bias is not None:
        assert bias.shape == (n,) and bias.dtype in _DTYPES, (
            "bias must be [n], bfloat16, float16 or float32")
        bias = bias.contiguous()
        bias_ptr, bias_type = bias.data_ptr(), _DTYPES[bias.dtype]
    if a.ndim != 2:
        a = a.reshape(-1, k)
        a_scale = a_scale.reshape(-1, kb)
    m = a.shape[0]
    a, lda = _byte_rows(a, k)
    w, ldw = _byte_rows(w, k)
    as_row, as_col = a_scale.stride()
    if as_row > _MAX_SCALE_STRIDE and m > 1:
        a_scale = a_scale.contiguous()
        as_row, as_col = kb, 1
    w_scale = w_scale.contiguous()
    if not given:
        out = a_scale.new_empty(lead + (n,), dtype=out_dtype)
    ldo = out.stride(0) if given and out.ndim == 2 else n
    _call(index, "fp8_block_matmul", _capi.load().fgs_moe_fp8_block_matmul,
          a.data_ptr(), lda, a_scale.data_ptr(), as_row, as_col, w.data_ptr(), ldw,
          w_scale.data_ptr(), bias_ptr, bias_type, m, n, k, _DTYPES[out_dtype], _flags,
          out.data_ptr(), ldo, _stream_ptr(a))
    if given:
        _written(out)
    return out


__all__ = [
    "fused_rms_norm",
    "silu_and_mul_quant",
    "fp8_block_matmul",
]
