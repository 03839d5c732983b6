"""The fast division by a row's scale (csrc/quant_ops.h) and the E4M3 codes of unrounded binary32 values, in exact
arithmetic."""

import random
from fractions import Fraction


def rounded(x):
    """To the nearest binary32, ties to even; nothing here overflows or underflows."""
    if x == 0:
        return x
    size = abs(x)
    e = size.numerator.bit_length() - size.denominator.bit_length()
    e -= Fraction(2) ** e > size
    n = size / Fraction(2) ** (e - 23)
    k, rest = divmod(n.numerator, n.denominator)
    k += 2 * rest + k % 2 > n.denominator
    return (k if x > 0 else -k) * Fraction(2) ** (e - 23)


def fast(x, s):
    y = rounded(1 / s)
    q0 = rounded(x * y)
    r = rounded(q0 * s - x)
    return rounded(q0 - r * y)


def test_rounding():
    for k, want in ((1 << 24, 1 << 24), ((1 << 24) + 1, 1 << 24), ((1 << 24) + 3, (1 << 24) + 4), ((1 << 25) + 3, (1 << 25) + 4)):
        assert rounded(Fraction(k)) == want and rounded(Fraction(-k, 1 << 40)) == Fraction(-want, 1 << 40)
    assert rounded(Fraction(1, 3)) == Fraction(11184811, 1 << 25)


def test_quotients_next_to_a_midpoint_of_e4m3():
    # All x and s whose fast and exact quotients could lie on two sides of a midpoint: s within 9 units of a multiple of
    # 1 / 8 (12 here), x nearest to (B +- half a unit of B) s, and its neighbours.
    unit, cases = Fraction(1, 1 << 23), 0
    for eighth in range(8, 17):
        for off in range(-12, 13):
            s = Fraction(eighth, 8) + off * unit
            if not 1 <= s < 2:
                continue
            for b in range(16, 33):
                for side in (-1, 1):
                    ulp = unit / 2 if b == 16 and side < 0 else 2 * unit if b == 32 and side > 0 else unit
                    x = rounded((Fraction(b, 16) + side * ulp / 2) * s)
                    for step in (-1, 0, 1):
                        near = x + step * (2 * unit if x >= 2 else unit)
                        assert fast(near, s) == rounded(near / s), (near, s)
                        cases += 1
    assert cases == 200 * 17 * 2 * 3


def test_random_quotients():
    rng = random.Random(1)
    for _ in range(5000):
        s = Fraction(rng.randrange(1 << 23, 1 << 24), 1 << 23)
        x = Fraction(rng.randrange(1 << 23, 1 << 24), 1 << rng.randrange(20, 36))
        assert fast(x, s) == rounded(x / s) and fast(-x, s) == -fast(x, s)
