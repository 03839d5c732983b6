"""Rotary phases against the frequencies that they were made of, at positions of any size, on the CPU."""

from fractions import Fraction

import pytest

from tests.rotary_reference import turns
from vflash_amd.rotary import Rotary, rotary_frequencies

POSITIONS = [0, 1, -1, 77, 131071, -1000003, 2**32, 2**40 + 3, -(2**50) - 1, 2**58 + 12345, 2**62 + 7, 2**63 - 1, -(2**63)]


@pytest.mark.parametrize("base", [10000.0, 5e5, 1e9])
def test_every_pair_at_every_position(base):
    frequencies = rotary_frequencies(128, base) + [3.75, -0.5, 1e-30, 12345.678]
    phases = Rotary(frequencies, device="cpu").phases.tolist()
    for f, phase in zip(frequencies, phases):
        for p in POSITIONS:
            # The kernel's product modulo 2^64, and the turns that the frequency says: half a step of 2^-64 a position.
            off = Fraction(p * phase % 2**64, 2**64) - turns(p, f)
            off -= round(off)
            assert abs(off) <= abs(p) * Fraction(1, 2**65) + Fraction(1, 2**120), (f, p)
