"""Tokens sorted by expert and back, for MI355X (gfx950).

A program that trains a routed layer, or sends its tokens to the GPUs that have
their experts, runs the layer in steps::

    weights, ids = fused_topk(x, logits, topk)
    rows, order = moe_permute(x, ids, num_experts)
    h = grouped_linear(rows, w13, order.counts, activation="silu", gated=True)
    out = moe_unpermute(grouped_linear(h, w2, order.counts), order, weights)

each with its gradients (the products are :mod:`flaggems_sglang.ops.linear`'s).
The host side is the extension module ``_host``; the arithmetic is in
``libfgs_moe.so`` (include/fgs_moe.h). There is no CPU path, no forward-mode
derivative and no second derivative.

The reference runs the layer as one call without gradients
(src/flaggems_sglang/ops/fused_moe.py:149-232); the order is that of its routing
conversion (:134-139) with a token's slots as they are given.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from flaggems_sglang import _capi
from flaggems_sglang.ops._autograd import needs_gradient

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


class ExpertOrder(NamedTuple):
    """The order that :func:`moe_permute` brings the tokens' slots (``topk`` each)
    into: by expert, within one by slot, the slots that no expert here has last."""

    counts: torch.Tensor  #: int32 ``[num_experts]``: rows of each expert
    row_of_slot: torch.Tensor  #: int32 ``[tokens, topk]``: -1 for slots without an expert
    slot_of_row: torch.Tensor  #: int32 ``[tokens * topk]``: -1 for the rows behind


def moe_permute(
    x: torch.Tensor,
    topk_ids: Optional[torch.Tensor] = None,
    num_experts: Optional[int] = None,
    *,
    order: Optional[ExpertOrder] = None,
) -> Tuple[torch.Tensor, ExpertOrder]:
    """The rows of ``x [tokens, cols]``, one for each of a token's ``topk`` slots,
    sorted by the slots' experts: ``rows[p] = x[slot_of_row[p] // topk]``,
    ``[tokens * topk, cols]``.

    ``topk_ids [tokens, topk]`` int32 or int64; ids outside ``[0, num_experts)``
    (experts of other GPUs) come behind the last expert's, as rows of zeros.
    ``num_experts`` up to 1022; up to 2^30 slots (gradients and rows by an ``order``:
    fewer than 2^23 tokens and 2^27 slots, else what their grids can hold). Or ``order``, as an earlier call
    on the same ids returned it: then nothing is sorted again (for the scales of
    8-bit values, say).

    ``x`` bf16, fp16 or fp32, or without gradients an 8-bit float or an 8-, 32- or
    64-bit integer type. ``x``'s gradient is the sum over a token's rows, in fp32 in
    the order of its slots. Returns ``(rows, ExpertOrder)``; nothing waits for the
    GPU.
    """
    if order is not None:
        if topk_ids is not None or num_experts is not None:
            raise ValueError("moe_permute: give topk_ids and num_experts, or an order")
    elif topk_ids is None or num_experts is None:
        raise ValueError("moe_permute: needs topk_ids and num_experts, or an order")
    elif topk_ids.dtype == torch.int64:  # (ids past 32 bits stay outside)
        topk_ids = topk_ids.clamp(-1, num_experts).to(torch.int32)
    with_grad = needs_gradient("moe_permute", x)
    if with_grad:
        assert x.dtype in _FLOATS, "x with a gradient must be bfloat16, float16 or float32"
    if order is not None:
        return _capi.host().permute_rows(x, order.row_of_slot, order.slot_of_row, with_grad), order
    rows, *made = _capi.host().permute(x, topk_ids, num_experts, with_grad)
    return rows, tuple.__new__(ExpertOrder, made)


def moe_unpermute(
    rows: torch.Tensor,
    order: ExpertOrder,
    topk_weights: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """The experts' results ``rows [tokens * topk, cols]`` (bf16, fp16 or fp32), in
    the ``order`` that :func:`moe_permute` returned, back to tokens::

        out[t] = sum_k topk_weights[t, k] * rows[order.row_of_slot[t, k]]

    in fp32 from k = 0 on, rounded once. ``topk_weights [tokens, topk]``: of any
    float type (taken in fp32), or None for ones. Slots without an expert add
    nothing, whatever their weight is and the rows behind hold.

    Gradients go to ``rows`` (zeros behind the experts' rows) and to
    ``topk_weights`` (summed in fp32).
    """
    assert rows.shape[0] == order.slot_of_row.shape[0], "the order is one of other rows"
    with_grad = needs_gradient("moe_unpermute", rows, topk_weights)  # (of the caller's tensors)
    if topk_weights is not None and topk_weights.dtype != torch.float32:
        topk_weights = topk_weights.float()
    return _capi.host().unpermute(rows, order.row_of_slot, order.slot_of_row, topk_weights, with_grad)


__all__ = [
    "moe_permute",
    "moe_unpermute",
]
