"""What the operators with gradients share."""

from __future__ import annotations

import torch

from flaggems_sglang import _capi


def needs_gradient(what, *tensors) -> bool:
    """Whether a gradient is to be recorded for one of the tensors (None: not given).

    While the current stream is captured into a graph, refuses a leaf whose
    gradient node an eager graph of another stream keeps alive: the captured
    backward pass would have that stream wait for the captured one, which breaks
    the capture off and ends the process.
    """
    if not torch.is_grad_enabled():
        return False
    need = False
    for t in tensors:
        if getattr(t, "requires_grad", False):  # (what is no tensor is refused later)
            need = True
    if need and torch.cuda.is_current_stream_capturing():
        for t in tensors:
            if isinstance(t, torch.Tensor) and _capi.host().foreign_leaf(t):
                raise RuntimeError(
                    f"{what}: an earlier graph of this leaf, recorded on another stream, is still "
                    "alive: its backward pass cannot be captured (delete that graph's outputs, or "
                    "record it on the stream that captures)")
    return need
