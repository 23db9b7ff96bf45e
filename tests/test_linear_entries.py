"""Refusals of the products' gradients' entries: no GPU is touched."""

import pytest

from flaggems_sglang import _capi
from test_steps import DW, DX, call


@pytest.mark.parametrize("name, defaults, which, forms", [
    ("linear_weight_grad", DW, "ldz", "weight"), ("linear_weight_grad", DW, "ldx", "weight"),
    ("linear_input_grad", DX, "ldw", "input")])
def test_rows_that_overlap(name, defaults, which, forms):
    """An operand whose sums run across its rows: less than its width apart."""
    for form in range(_capi.LINEAR_FORMS[forms] + 1):
        for ld in (0, 8, defaults[which] - 8):
            rc, text = call(name, defaults, **{which: ld, "flags": form})
            assert rc == -2 and "overlap" in text, text
