"""Rotary tables' arguments (no GPU)."""

import pytest

from browservec_amd import _lib as L
from browservec_amd import rotary_table


def test_a_magnitude_of_zero_is_refused():
    """The library's 0 means 1."""
    for magnitude in (0, 0.0, -0.0):
        with pytest.raises(L.BVError) as e:
            rotary_table(4, 8, magnitude=magnitude)
        assert e.value.code == L.BV_E_INVALID
    assert rotary_table(4, 8, magnitude=-2.0)[0, 0, 0] == -2.0
