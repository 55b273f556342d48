"""Attention over the paged cache: caps whose reciprocal leaves fp32 are refused on the host."""
import pytest

from test_paged_arguments_cpu import attend


@pytest.mark.parametrize("cap", [1e-45, 1e-39, 9e-31, 2e30])
def test_caps_without_a_reciprocal(cap):
    """1 / softcap is infinite below 2^-128, and a score of zero would become NaN."""
    assert attend(cap=cap) == -1


@pytest.mark.parametrize("cap", [0.0, 1e-30, 30.0, 1e30])
def test_caps_that_are_taken(cap):
    assert attend(cap=cap, tokens=0) == 0
