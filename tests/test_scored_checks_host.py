"""More that scored attention and the 4-bit pool refuse, without a GPU."""

from __future__ import annotations

import pytest

from memforge_amd import _native as nat


@pytest.mark.parametrize("cap", [1e-50, 1e39, -1e-50])
def test_caps_that_32_bits_do_not_hold(cap):
    """1e-50 is 0 in 32 bits: no cap at all instead of one that flattens every score."""
    with pytest.raises(ValueError):
        nat.Scoring(cap)
