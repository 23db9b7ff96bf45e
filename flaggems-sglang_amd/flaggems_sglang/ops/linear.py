"""Products of 16-bit matrices with bias, activation and residual in the epilogue,
and their gradients, for MI355X (gfx950).

:func:`fused_linear` is a layer's dense product (the shared expert's, the
projections'), :func:`grouped_linear` that of the experts with rows sorted by
expert (:mod:`flaggems_sglang.ops.steps`). The host side is the extension module
``_host``; the arithmetic is in ``libfgs_moe.so`` (include/fgs_moe.h). There is no
CPU path, no forward-mode derivative and no second derivative.

The reference's products (matmul_ogs, src/flaggems_sglang/ops/fused_moe.py:205-231)
have neither a dense form nor gradients.
"""

from __future__ import annotations

from typing import Optional

import torch

from flaggems_sglang import _capi
from flaggems_sglang.ops._autograd import needs_gradient

_ACTIVATIONS = {None: _capi.ACT_NONE, "relu": _capi.ACT_RELU, "silu": _capi.ACT_SILU,
                "gelu": _capi.ACT_GELU}


def _linear(what, x, weight, counts, bias, activation, gated, residual, flags):
    act = _ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"Unsupported activation: {activation}")
    return _capi.host().linear(x, weight, counts, bias, act, gated, residual,
                               needs_gradient(what, x, weight, bias, residual), flags)


def fused_linear(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    *,
    activation: Optional[str] = None,
    gated: bool = False,
    residual: Optional[torch.Tensor] = None,
    _flags: int = 0,
) -> torch.Tensor:
    """``activation(x @ weight.T + bias) + residual``, or with ``gated`` and
    ``weight = [gate rows | up rows]``::

        activation(x @ gate.T + bias_gate) * (x @ up.T + bias_up) + residual

    ``x [..., k]``, ``weight [n, k]`` (gated: ``[2 n, k]``), ``bias`` of weight's
    first size, ``residual [..., n]``, all bf16 or all fp16. Sums, activation and
    additions are in fp32, the result is rounded once. ``activation``: None,
    "relu", "silu" or "gelu" (exact, erf). ``n`` and ``k`` are multiples of 8 up to
    2^20 (gated: ``2 n``); fewer than 2^30 rows (0 among them). Operands whose rows are not 16-byte
    aligned, or whose columns are not adjacent, are copied first, and by the gradients
    those whose rows overlap (broadcast rows, sliding windows).

    Gradients go to ``x``, ``weight``, ``bias`` and ``residual``. With an activation,
    what it is taken of is kept in fp32 for them, and its gradient is rounded to x's
    type, in which x's and the weight's products take it; the bias's sums take what
    that rounding leaves as well.
    """
    return _linear("fused_linear", x, weight, None, bias, activation, gated, residual, _flags)


def grouped_linear(
    x: torch.Tensor,
    weight: torch.Tensor,
    counts: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    *,
    activation: Optional[str] = None,
    gated: bool = False,
    residual: Optional[torch.Tensor] = None,
    _flags: int = 0,
) -> torch.Tensor:
    """:func:`fused_linear` with a matrix for each group of rows: ``x [rows, k]``
    sorted by group, ``weight [groups, n, k]`` (gated: ``2 n``), ``counts [groups]``
    int32 on the GPU (``moe_permute``'s), ``bias [groups, n]``, ``residual [rows,
    n]``; up to 4096 groups. Group ``e`` has the ``counts[e]`` rows behind those of
    the groups before it (a negative count is 0; counts past the last row are cut).
    Rows behind the last group's have no product: zeros, or the residual's, and no
    gradient but its. An empty group's weight has a gradient of zeros.
    """
    if counts is None:
        raise TypeError("counts must be a tensor")
    return _linear("grouped_linear", x, weight, counts, bias, activation, gated, residual, _flags)


__all__ = [
    "fused_linear",
    "grouped_linear",
]
