"""How good the rotary frequencies and, from them, far angles are, against
60-digit arithmetic; no device needed."""
from decimal import Decimal, getcontext

import pytest

attention = pytest.importorskip("pspml.attention")
getcontext().prec = 60
TWO_PI = 2 * Decimal("3.14159265358979323846264338327950288419716939937510582097494459")


@pytest.mark.parametrize("rot,base,factor", [(128, 10000.0, 1.0), (64, 500000.0, 1.0),
                                             (6, 3.5, 1.0), (128, 1000000.0, 8.0)])
def test_angles_at_far_positions(rot, base, factor):
    # A power, a quotient by the factor and one by 2 pi, each rounded to 53 bits (the power to an
    # ulp or so): 2^-51 of a frequency is room enough, and a position multiplies it.
    bits = attention.rotary_frequencies(attention.rotary_desc(
        rot, base=base, scaling="linear" if factor != 1.0 else "none", factor=factor))
    for i, b in enumerate(bits):
        turns = (-Decimal(2 * i) / rot * Decimal(base).ln()).exp() / Decimal(factor) / TWO_PI
        off = abs(Decimal(int(b)) / 2 ** 64 - turns)
        assert off <= turns / 2 ** 51 + Decimal(2) ** -64
    # What the interface says of the fastest pair at position 2^31.
    if factor == 1.0:
        assert abs(Decimal(int(bits[0])) / 2 ** 64 - 1 / TWO_PI) * 2 ** 31 <= Decimal(2) ** -24
