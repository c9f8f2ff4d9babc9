"""Refusals of the paged memory's operators at the ends of what an argument may be."""
import pytest

import sarbon_b200 as sb
from test_paged_ops_cpu import EVICT


@pytest.mark.parametrize("keep", [float("inf"), float("nan"), -float("inf"), -1, 0.5, 7.25])
def test_budgets_that_are_no_whole_number(keep):
    with pytest.raises(ValueError, match="whole number"):
        sb.paged_evict(**{**EVICT, "keep": keep})
