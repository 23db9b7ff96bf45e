"""Which tensors are looked at before a captured call records a graph (the host module
replaced: no GPU is touched)."""

import pytest
import torch

import flaggems_sglang as fgs
from flaggems_sglang import _capi
from flaggems_sglang.ops import fused_moe, steps

X = torch.ones(4, 64, dtype=torch.bfloat16)


class Host:
    """Every leaf has a graph of another stream."""

    def __init__(self):
        self.asked = []

    def foreign_leaf(self, t):
        self.asked.append(t)
        return t.requires_grad and t.is_leaf

    def unpermute(self, *args):
        raise AssertionError("a graph was recorded")

    topk_gating = unpermute


@pytest.fixture
def host(monkeypatch):
    h = Host()
    monkeypatch.setattr(_capi, "_host", h)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    monkeypatch.setattr(fused_moe, "_require_gpu", lambda *a: None)
    return h


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.float64])
def test_leaves_of_other_types(host, dtype):
    """The caller's own tensor, not a copy in another type that is no leaf."""
    order = steps.ExpertOrder(torch.zeros(3, dtype=torch.int32), torch.zeros(4, 2, dtype=torch.int32),
                              torch.zeros(8, dtype=torch.int32))
    logits = torch.ones(4, 8, dtype=dtype, requires_grad=True)
    weights = torch.ones(4, 2, dtype=dtype, requires_grad=True)
    for call, leaf in ((lambda: fgs.fused_topk(X, logits, 2), logits),
                       (lambda: fgs.moe_unpermute(X.repeat(2, 1), order, weights), weights)):
        with pytest.raises(RuntimeError, match="still alive"):
            call()
        assert host.asked[-1] is leaf
