"""The angles of rotary positions from the frequencies themselves, as rationals."""

from fractions import Fraction

import torch

# 2 pi to 60 digits: a position of 2^63 turns of it are known to 2^-130.
TURN = Fraction("6.28318530717958647692528676655900576839433879875021164194989")


def turns(position, frequency):
    """The turns of a position modulo one, in [-1/2, 1/2)."""
    t = Fraction(int(position)) * Fraction(frequency) / TURN + Fraction(1, 2)
    return t - t.__floor__() - Fraction(1, 2)


def angles(positions, frequencies):
    """Radians, [positions, pairs], and how far the kernel's may be from them."""
    angle = torch.tensor([[float(turns(p, f) * TURN) for f in frequencies] for p in positions], dtype=torch.float64)
    off = torch.tensor([float(TURN) * (2.0**-33 + abs(int(p)) * 2.0**-65) for p in positions], dtype=torch.float64)
    return angle, off[:, None].expand_as(angle)
