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
_GROUP = 128  # columns of an e4m3 scale


class RMSNormOutput(NamedTuple):
    """What :func:`fused_rms_norm` returns; what a call does not make is None."""

    norm: Optional[torch.Tensor]
    residual: Optional[torch.Tensor]
    q: Optional[torch.Tensor]
    scales: Optional[torch.Tensor]


def _check_inputs(**tensors) -> torch.device:
    """Every tensor given is on one GPU and needs no gradient; that GPU."""
    device = None
    grad = torch.is_grad_enabled()
    for name, t in tensors.items():
        if t is None:
            continue
        if device is None:
            _require_gpu(name, t)
            device = t.device
        elif t.device != device:
            raise RuntimeError(f"{name} is on {t.device}, not on {device}")
        if grad and t.requires_grad:
            raise RuntimeError(f"{name} requires a gradient: this operator has no backward "
                               "pass (call it under torch.no_grad())")
    return device


def _call(device: torch.device, fn, what: str, *args) -> None:
    """Runs a library entry on ``device`` (whichever device is current)."""
    if device.index == torch.cuda.current_device():
        rc = fn(*args)
    else:
        with torch.cuda.device(device):
            rc = fn(*args)
    _capi.check(rc, what)


def _written(t: torch.Tensor) -> None:
    """Tells autograd that the library has written a caller's tensor."""
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)


def _rows(x: torch.Tensor):
    """``x`` as rows of its last dimension: (tensor whose storage they are in,
    number of rows, row stride in elements). Rows that lie evenly spaced, as
    those of a slice of a wider tensor, are taken where they are."""
    cols = x.shape[-1]
    if x.ndim == 2:
        if x.stride(1) == 1 or cols == 1:
            return x, x.shape[0], x.stride(0)
    elif x.is_contiguous():
        return x, x.numel() // cols, cols
    x = x.contiguous()
    return x, x.numel() // cols, cols


def _quant_outputs(shape, rows: int, cols: int, quant: int, column_major: bool,
                   device: torch.device):
    """``(q, scales, stride of the scales over rows, over groups)``."""
    if quant == _capi.QUANT_NONE:
        return None, None, 0, 0
    if quant == _capi.QUANT_INT8_TOKEN:
        q = torch.empty(shape, dtype=torch.int8, device=device)
        return q, torch.empty(shape[:-1], dtype=torch.float32, device=device), 1, 0
    groups = (cols + _GROUP - 1) // _GROUP
    q = torch.empty(shape, dtype=torch.float8_e4m3fn, device=device)
    if not column_major:
        scales = torch.empty(shape[:-1] + (groups,), dtype=torch.float32, device=device)
        return q, scales, groups, 1
    scales = torch.empty((groups, rows), dtype=torch.float32, device=device).t()
    if len(shape) != 2:
        scales = scales.view(shape[:-1] + (groups,))
    return q, scales, 1, rows


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
    device = _check_inputs(x=x, weight=weight, residual=residual)
    if quant not in _QUANTS:
        raise ValueError(f"Unsupported quantisation: {quant}")
    assert x.dtype in _DTYPES, "x must be bfloat16, float16 or float32"
    assert x.ndim >= 1 and x.shape[-1] > 0, "x must have columns"
    cols = x.shape[-1]
    assert weight.shape == (cols,), "weight must be [cols]"
    assert weight.dtype in (x.dtype, torch.float32), "weight must be of x's type or float32"
    if return_norm is None:
        return_norm = quant is None
    assert return_norm or quant is not None or residual is not None, "no output was asked for"
    assert not inplace or residual is not None, "inplace needs a residual"
    mode = _QUANTS[quant]
    shape = tuple(x.shape)
    xr, rows, x_stride = _rows(x)
    rr = res_out = None
    r_stride = out_stride = 0
    if residual is not None:
        assert residual.shape == x.shape and residual.dtype == x.dtype, (
            "residual must be of x's shape and type")
        rr, _, r_stride = _rows(residual)
        if inplace:
            if rr is not residual or (rows > 1 and r_stride < cols):
                raise ValueError("fused_rms_norm: an inplace residual must have evenly spaced "
                                 "rows that do not overlap")
            res_out, out_stride = residual, r_stride
        else:
            res_out = torch.empty(shape, dtype=x.dtype, device=device)
            out_stride = cols
    norm = torch.empty(shape, dtype=x.dtype, device=device) if return_norm else None
    q, scales, s_row, s_col = _quant_outputs(shape, rows, cols, mode, column_major_scales, device)
    weight = weight.contiguous()
    _call(device, _capi.load().fgs_moe_rms_norm, "fused_rms_norm",
          xr.data_ptr(), x_stride, None if rr is None else rr.data_ptr(), r_stride,
          weight.data_ptr(), _DTYPES[x.dtype], _DTYPES[weight.dtype], eps, weight_offset, rows,
          cols, None if norm is None else norm.data_ptr(),
          None if res_out is None else res_out.data_ptr(), out_stride, mode,
          None if q is None else q.data_ptr(), None if scales is None else scales.data_ptr(),
          s_row, s_col, _stream_ptr(x))
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
    device = _check_inputs(x=x)
    if activation not in ("silu", "gelu"):
        raise ValueError(f"Unsupported activation: {activation}")
    if quant is None or quant not in _QUANTS:
        raise ValueError(f"Unsupported quantisation: {quant}")
    assert x.dtype in _DTYPES, "x must be bfloat16, float16 or float32"
    assert x.ndim >= 1 and x.shape[-1] % 2 == 0 and x.shape[-1] > 0, (
        "x must hold a gate half and an up half")
    n = x.shape[-1] // 2
    mode = _QUANTS[quant]
    xr, rows, x_stride = _rows(x)
    q, scales, s_row, s_col = _quant_outputs(tuple(x.shape[:-1]) + (n,), rows, n, mode,
                                             column_major_scales, device)
    _call(device, _capi.load().fgs_moe_silu_and_mul_quant, "silu_and_mul_quant",
          xr.data_ptr(), x_stride, _DTYPES[x.dtype], rows, n, 1 if activation == "gelu" else 0,
          mode, q.data_ptr(), scales.data_ptr(), s_row, s_col, _stream_ptr(x))
    return q, scales


def _byte_rows(t: torch.Tensor):
    """An e4m3 matrix with adjacent columns and 16-byte aligned rows, and its
    row stride: where it is, or copied."""
    if (t.stride(1) == 1 and (t.shape[0] <= 1 or t.stride(0) % 16 == 0)
            and t.data_ptr() % 16 == 0):
        return t, t.stride(0)
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.shape[1]


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
    device = _check_inputs(a=a, a_scale=a_scale, w=w, w_scale=w_scale, bias=bias, out=out)
    assert a.dtype == torch.float8_e4m3fn and w.dtype == torch.float8_e4m3fn, (
        "a and w must be float8_e4m3fn")
    assert w.ndim == 2 and a.ndim >= 1 and a.shape[-1] == w.shape[1], (
        "a must be [..., k] and w [n, k]")
    n, k = w.shape
    lead = tuple(a.shape[:-1])
    kb = (k + _GROUP - 1) // _GROUP
    assert tuple(a_scale.shape) == lead + (kb,), "a_scale must be [..., ceil(k / 128)]"
    assert tuple(w_scale.shape) == ((n + _GROUP - 1) // _GROUP, kb), (
        "w_scale must be [ceil(n / 128), ceil(k / 128)]")
    assert a_scale.dtype == torch.float32 and w_scale.dtype == torch.float32, (
        "scales must be float32")
    if out is not None:
        out_dtype = out.dtype
        assert tuple(out.shape) == lead + (n,), "out must be [..., n]"
        if out.stride(-1) != 1 if out.ndim == 2 else not out.is_contiguous():
            raise ValueError("fp8_block_matmul: the columns of out must be adjacent")
    assert out_dtype in (torch.bfloat16, torch.float16), "the output must be bfloat16 or float16"
    if bias is not None:
        assert bias.shape == (n,) and bias.dtype in _DTYPES, (
            "bias must be [n], bfloat16, float16 or float32")
        bias = bias.contiguous()
    if a.ndim != 2:
        a = a.reshape(-1, k)
        a_scale = a_scale.reshape(-1, kb)
    m = a.shape[0]
    ar, lda = _byte_rows(a)
    wr, ldw = _byte_rows(w)
    w_scale = w_scale.contiguous()
    given = out is not None
    if not given:
        out = torch.empty(lead + (n,), dtype=out_dtype, device=device)
    ldo = out.stride(0) if out.ndim == 2 else n
    lib = _capi.load()
    ws_bytes = lib.fgs_moe_fp8_block_matmul_workspace_bytes(m, n, k, _flags)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device) if ws_bytes > 0 else None
    _call(device, lib.fgs_moe_fp8_block_matmul, "fp8_block_matmul",
          ar.data_ptr(), lda, a_scale.data_ptr(), a_scale.stride(0), a_scale.stride(1),
          wr.data_ptr(), ldw, w_scale.data_ptr(), None if bias is None else bias.data_ptr(),
          _DTYPES[out_dtype] if bias is None else _DTYPES[bias.dtype], m, n, k,
          _DTYPES[out_dtype], _flags, None if ws is None else ws.data_ptr(), max(ws_bytes, 0),
          out.data_ptr(), ldo, _stream_ptr(a))
    if given:
        _written(out)
    return out


__all__ = [
    "fused_rms_norm",
    "silu_and_mul_quant",
    "fp8_block_matmul",
]
