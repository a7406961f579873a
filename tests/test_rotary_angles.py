"""The frequencies of ``AxialRotary`` as 64-bit fractions of a turn (no GPU)."""

from decimal import Decimal, localcontext

import pytest

from recap_b200 import AxialRotary


@pytest.mark.parametrize("ladder", ["axis", "shared"])
@pytest.mark.parametrize("scale", [1.0, 0.37, 2.5, 1e-6, 12345.678])
def test_a_negative_scale_turns_back_by_the_same_angle(scale, ladder):
    dims = (16, 24, 24)
    forth, back = (AxialRotary(64, dims, theta=10000.0, ladder=ladder, scale=s) for s in (scale, -scale))
    n = forth._struct.pairs
    assert [t % 2**64 for t in back._struct.turns[:n]] == [-t % 2**64 for t in forth._struct.turns[:n]]


PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494459")


@pytest.mark.parametrize("theta", [1.5, 256.0, 10000.0, 12345.678, 1e6])
@pytest.mark.parametrize("ladder", ["axis", "shared"])
@pytest.mark.parametrize("scale", [1.0, -1.0, 0.3, 7.1])
def test_frequencies_against_the_definition_in_60_digits(theta, ladder, scale):
    """With u = 2^-53 and x the exponent: rounding x moves theta ** -x by ln(theta) x u of itself, the power adds 2 u,
    2 pi and the division 1.4 u, the scale u.  Times the frequency theta ** -x / (2 pi), at most (v + 4.4) e^-v / (2 pi)
    with v = ln(theta) x, that is under u for every theta of 1 or more; the 64 bits add 2^-65."""
    with localcontext() as context:
        context.prec = 60
        for dims in ((8,), (44, 42, 42), (128,), (64, 64, 64, 64)):
            r = AxialRotary((sum(dims) + 7) // 8 * 8, dims, theta=theta, ladder=ladder, scale=scale)
            exponents = [Decimal(2 * p) / sum(dims) for p in range(sum(dims) // 2)] if ladder == "shared" else \
                [Decimal(2 * i) / d for d in dims for i in range(d // 2)]
            for turns, x in zip(r._struct.turns, exponents):
                want = (-x * Decimal(theta).ln()).exp() / (2 * PI) * Decimal(scale) * 2**64
                off = (Decimal(turns) - want + 2**63) % 2**64
                off = abs((off + 2**64 if off < 0 else off) - 2**63)
                assert off <= abs(Decimal(scale)) * 2**11 + Decimal("0.5")
