"""Refusals of the steps' gradients' entries: no GPU is touched."""

import pytest

from flaggems_sglang import _capi
from test_steps import ACT, DB, DW, DX, TOPK, call


@pytest.mark.parametrize("name, defaults, which, forms", [
    ("linear_weight_grad", DW, "ldz", "weight"), ("linear_weight_grad", DW, "ldx", "weight"),
    ("linear_input_grad", DX, "ldw", "input")])
def test_rows_that_overlap(name, defaults, which, forms):
    """An operand whose sums run across its rows: less than its width apart."""
    for form in range(_capi.LINEAR_FORMS[forms] + 1):
        for ld in (0, 8, defaults[which] - 8):
            rc, text = call(name, defaults, **{which: ld, "flags": form})
            assert rc == -2 and "overlap" in text, text


@pytest.mark.parametrize("scoring, renorm", [(0, 0), (1, 1)])
def test_logits_that_are_read(scoring, renorm):
    rc, text = call("topk_gating_grad", TOPK, logits=None, scoring=scoring, renorm=renorm)
    assert rc == -1 and "null pointer" in text, text


def test_rests_lie_behind_contiguous_rows():
    rc, text = call("linear_bias_grad", DB, ldz=40, dtype=0x100)
    assert rc == -1 and "contiguous" in text, text
    for name, defaults in (("linear_act_grad", ACT), ("linear_bias_grad", DB)):
        rc, text = call(name, defaults, dtype=0x102)
        assert rc == -2 and "bf16 or fp16" in text, text
