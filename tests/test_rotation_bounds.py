"""The bounds that the head rotation states for its angles, sines and cosines (mq_heads.hip, moldq.h),
on the CPU: its formulas with the numbers that its source has, against exact fractions and
extended precision.  An extended result that stands for a fused multiply-add is rounded twice, 2^-12 of
a 64-bit last place more, nothing beside 2^-29."""
import pathlib
import random
import re
from fractions import Fraction

import numpy as np
import pytest

SOURCE = (pathlib.Path(__file__).parent.parent / "mold_amd" / "csrc" / "mq_heads.hip").read_text()
L = np.longdouble
PI = Fraction(31415926535897932384626433832795028841971693993751, 10 ** 49)


def test_angles():
    """position * (inv_freq * 1 / (2 pi)): the constant and two products, each within 2^-53 of itself, of 2^28.35
    turns at most: 3 * 2^-24.65 < 2^-23."""
    turn = float(re.search(r"freq\[i\] = \(double\)v\[i\] \* ([0-9.]+);", SOURCE).group(1))
    off = abs(Fraction(turn) * 2 * PI - 1) * 2 ** 53
    assert (2 + off) * Fraction(2 ** 31) / (2 * PI) / 2 ** 53 < Fraction(1, 2 ** 23)
    rng = random.Random(0)
    for i in range(20000):
        position = (1 << 31) - rng.randrange(1 << 20) if i % 2 else rng.randrange(1 << 31)
        freq = float(np.float32(rng.uniform(0.5, 1.0)))
        assert abs(Fraction(position * (freq * turn)) - position * Fraction(freq) / (2 * PI)) < Fraction(1, 2 ** 23)


@pytest.mark.skipif(np.finfo(L).nmant < 63, reason="no extended precision")
def test_sine_and_cosine():
    lines = SOURCE[SOURCE.index("double x = __builtin_fma(z,"):SOURCE.index("const float sine")]
    numbers = [float(n) for n in re.findall(r"-?[0-9]+\.[0-9]+", lines)]
    assert len(numbers) == 10
    r = np.random.default_rng(0).uniform(-0.125, 0.125, 1 << 20)
    r[:5] = 0.125, -0.125, 0.0, 1e-9, -1e-300
    z = r * r

    def fma(a, b, c):
        return (a.astype(L) * b + L(c)).astype(np.float64)
    x = fma(z, numbers[0], numbers[1])
    for n in numbers[2:5]:
        x = fma(z, x, n)
    y = fma(z, numbers[5], numbers[6])
    for n in numbers[7:]:
        y = fma(z, y, n)
    turn = 8 * np.arctan(L(1))
    for got, want, ulps, rest in ((r * x, np.sin(turn * r), 0.53, 2.0 ** -29), (fma(z, y, 1.0), np.cos(turn * r), 0.51, 2.0 ** -32)):
        assert np.abs(got.astype(L) - want).max() <= rest
        assert (np.abs(got.astype(np.float32).astype(L) - want) <= ulps * np.spacing(np.abs(want).astype(np.float32))).all()
