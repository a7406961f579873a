"""The frequencies of ``AxialRotary`` as 64-bit fractions of a turn (no GPU)."""

import pytest

from recap_b200 import AxialRotary


@pytest.mark.parametrize("ladder", ["axis", "shared"])
@pytest.mark.parametrize("scale", [1.0, 0.37, 2.5, 1e-6, 12345.678])
def test_a_negative_scale_turns_back_by_the_same_angle(scale, ladder):
    dims = (16, 24, 24)
    forth, back = (AxialRotary(64, dims, theta=10000.0, ladder=ladder, scale=s) for s in (scale, -scale))
    n = forth._struct.pairs
    assert [t % 2**64 for t in back._struct.turns[:n]] == [-t % 2**64 for t in forth._struct.turns[:n]]
