"""The rotation's angles against exact ones: the product of position and frequency as integers, reduced by 90 digits of pi.  The
kernel's angle is that product rounded to f64, off by 2^-53 of itself.

U = 2^-24 is half an f32 step relative to the value."""
import math
from fractions import Fraction

import numpy as np
import pytest

from attention_ref import U
from gpu_util import device
from test_gpu_lm_attention import blank, get, rotation, up

pytestmark = pytest.mark.gpu

PI = Fraction(314159265358979323846264338327950288419716939937510582097494459230781640628620899862803482, 10 ** 89)


def exact_turn(pos, f):
    """cos and sin of pos * f."""
    a = Fraction(int(pos)) * Fraction(float(np.float32(f)))
    r = a - 2 * PI * round(a / (2 * PI))  # within half a turn: as an f64 it is off by 2^-53 of itself
    return math.cos(r), math.sin(r)


@pytest.mark.parametrize("pairs", [False, True])
def test_angles_of_more_than_53_bits(pairs):
    d = device()
    pos = np.array([-(1 << 31), -(1 << 31) + 1, -1999999999, -70001, -1, 0, 1, 16777217, 1234567891, (1 << 31) - 19, (1 << 31) - 2, (1 << 31) - 1], np.int64)
    freq = np.float32([1.0, 0.99999994, 3.1415927, 3.14, 2.7182817, 1.5707964, 0.7853982, 0.33333334, 100.3, 777.77, 12345.678, 1.0e6] + [0.1234567 * 1.37 ** i for i in range(52)])
    x = np.zeros((len(pos), 1, 128), np.float32)
    first, second = (slice(0, 128, 2), slice(1, 128, 2)) if pairs else (slice(0, 64), slice(64, 128))
    x[..., first] = 1.0
    y = blank(len(pos), 128)
    d.rotate_heads(len(pos), 1, 128, y, up(x), rotation=rotation(pos, freq, 128, pairs))
    got = get(y, len(pos), 128).astype(np.float64)
    want = np.array([[exact_turn(p, f) for f in freq] for p in pos])
    angle = np.abs(np.outer(pos.astype(np.float64), freq.astype(np.float64)))
    # the reduced angle as an f32 and what it loses (first order: its square is below an f32 step of the result), sine or cosine to 2 steps
    # (4 U), the correction's sum and two products; the angle's own rounding
    assert np.all(np.abs(got[:, first] - want[..., 0]) <= 8 * U + 2.0 ** -53 * angle)
    assert np.all(np.abs(got[:, second] - want[..., 1]) <= 8 * U + 2.0 ** -53 * angle)
