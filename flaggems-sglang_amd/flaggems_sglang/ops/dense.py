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

The host side (checks of the arguments, allocation of the outputs with the
torch caching allocator, the call on the current HIP stream of the tensors'
GPU) is the extension module ``_host``; the arithmetic is in
``libfgs_moe.so`` (include/fgs_moe.h). There is no CPU path. None of these
has a backward pass or a forward-mode derivative: an input that requires a
gradient is refused while gradients are recorded, and so is a dual tensor of
``torch.autograd.forward_ad``.

The reference's fused-MoE path has no counterparts (its layer takes its input
normalised, and src/flaggems_sglang/ops/fused_moe.py:170-185 rejects every
8-bit mode).
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from flaggems_sglang import _capi

_OUT_DTYPES = {torch.bfloat16: _capi.DTYPE_BF16, torch.float16: _capi.DTYPE_FP16}
_QUANTS = {None: _capi.QUANT_NONE, "fp8": _capi.QUANT_FP8_GROUP,
           "int8": _capi.QUANT_INT8_TOKEN}
_ACTIVATIONS = {"silu": False, "gelu": True}


class RMSNormOutput(NamedTuple):
    """What :func:`fused_rms_norm` returns; what a call does not make is None."""

    norm: Optional[torch.Tensor]
    residual: Optional[torch.Tensor]
    q: Optional[torch.Tensor]
    scales: Optional[torch.Tensor]


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
    ``weight_offset=1`` for weights stored about zero. ``cols`` from 1 to 65536;
    multiples of 8 with 16-byte aligned rows run fastest (4096 x 7168 bf16 with
    four outputs 45 us, x 7167 163). Fewer than 2^22 rows, of few columns more.

    ``quant="fp8"``: ``q`` e4m3fn with ``scales [..., ceil(cols / 128)]`` per
    128 columns, ``"int8"``: ``q`` int8 with ``scales [...]`` per row (the
    codes of ``per_token_group_quant_fp8`` / ``per_token_quant_int8``, here of
    the unrounded ``n``). ``column_major_scales`` lays e4m3 scales out with
    the rows adjacent, which :func:`fp8_block_matmul` reads faster from some
    dozens of rows on. ``return_norm``: whether ``n`` comes back in x's type
    (default: where nothing is quantised). ``inplace``: the sum replaces
    ``residual``'s values and ``residual`` is the residual output (``x`` may be
    ``residual`` itself; an ``x`` or ``weight`` that shares its memory otherwise
    is refused).

    A NaN in a row makes its outputs NaN (int8 codes 0, scale NaN); a row whose
    squares sum past fp32's range (values of about 1e19) becomes zeros. Returns
    ``RMSNormOutput(norm, residual, q, scales)``.
    """
    mode = _QUANTS.get(quant)
    if mode is None:
        raise ValueError(f"Unsupported quantisation: {quant}")
    return tuple.__new__(RMSNormOutput, _capi.host().rms_norm(
        x, weight, eps, residual, weight_offset, mode, return_norm, column_major_scales, inplace))


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
    ``column_major_scales`` as for :func:`fused_rms_norm`; ``n`` from 1 to 65536
    (odd ones one value a load: 4096 x 7168 31 us, x 7167 71), rows as there.
    Returns ``(q [..., n], scales)``.
    """
    gelu = _ACTIVATIONS.get(activation)
    if gelu is None:
        raise ValueError(f"Unsupported activation: {activation}")
    mode = _QUANTS.get(quant)
    if not mode:
        raise ValueError(f"Unsupported quantisation: {quant}")
    return _capi.host().silu_and_mul_quant(x, mode, gelu, column_major_scales)


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
    :func:`silu_and_mul_quant` return, row- or column-major: with rows that lie
    apart a block's scales are a cache line each, 3 to 19 % more time from 64
    rows on), ``w [n, k]`` with ``w_scale [ceil(n / 128), ceil(k / 128)]``
    (``quant.quantize_fp8_block``). ``k`` is a multiple of 16 and ``n`` is at
    least 1; both and the number of rows (0 among them) go up to 2^22. Sums are
    fp32, of groups of eight products that the matrix instruction aligns to the
    largest and cuts 13 bits below it: about 1.5e-5 of a result from normal
    data, at most 7 * 2^-13 of each group's largest product, also where these
    cancel. The two scales are multiplied first, in fp32, whose range their
    product has to stay in. ``bias [n]`` (fp32, bf16 or fp16) is added to them, and the result is
    rounded once to ``out_dtype`` (bf16 or fp16). ``out``: a tensor of the
    result's shape to write and return, whose type counts instead of
    ``out_dtype``, whose rows may lie apart (2-D); one that shares memory with
    an input is refused.
    """
    code = _OUT_DTYPES.get(out_dtype, _capi.DTYPE_FP32)  # (refused there)
    return _capi.host().fp8_block_matmul(a, a_scale, w, w_scale, bias, code, out, _flags)


__all__ = [
    "fused_rms_norm",
    "silu_and_mul_quant",
    "fp8_block_matmul",
]
