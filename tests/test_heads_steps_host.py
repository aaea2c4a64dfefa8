"""How far a frequency's fraction of a turn is from the frequency, with pi to sixty digits, without a GPU.

The quotient f / (2 pi) is a double: math.pi is off by 2^-54 of pi, the quotient by 2^-53 of itself, the whole number of 2^-64 turns
by half of one.  Behind that nothing is lost: position times step is a product of whole numbers."""
import math
from fractions import Fraction

import pytest

from native_sparse_attention_pytorch_b200 import RotaryFrequencies

PI = Fraction('3.14159265358979323846264338327950288419716939937510582097494459')


@pytest.mark.parametrize('kwargs', [dict(), dict(theta=500000.0), dict(scaling='linear', factor=8.0), dict(scaling='ntk', factor=4.0),
                                    dict(scaling='yarn', factor=16.0, original_length=4096), dict(frequencies=[1.0, -0.125, 3.0, 1e-9] * 8)])
@pytest.mark.parametrize('position', [1, (1 << 20) + 3, 1 << 33, -(1 << 40)])
def test_angles_are_within_the_documented_bound(kwargs, position):
    rotary = RotaryFrequencies(64, **kwargs)
    for f, step in zip(rotary.frequencies, rotary._steps.tolist()):
        turns = Fraction(f) / (2 * PI)
        off = abs(Fraction(step % 2 ** 64, 2 ** 64) - turns) % 1
        assert min(off, 1 - off) <= abs(turns) * Fraction(1, 2 ** 52) + Fraction(1, 2 ** 65)
        # in radians, as documented: |position| (|f| 2^-52 + 2^-62)
        phase = Fraction(position * step % 2 ** 64, 2 ** 64)
        off = abs(phase - position * turns) % 1
        assert min(off, 1 - off) * 2 * PI <= abs(position) * (Fraction(abs(f)) / 2 ** 52 + Fraction(1, 2 ** 62))
    assert math.isfinite(rotary.magnitude)
