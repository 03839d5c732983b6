"""Rotary positions on the GPU against the frequencies themselves, at positions of any size."""

import pytest
import torch

from tests.rotary_reference import angles
from vflash_amd.rotary import Rotary, rotary_frequencies, rotate

pytestmark = pytest.mark.gpu
POSITIONS = [0, 1, -1, 1000003, (1 << 32) + 1, -(1 << 40) - 3, (1 << 50) + 1, -(1 << 58) - 5, (1 << 62) + 7, (1 << 63) - 1, -(1 << 63)]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("base", [1e4, 5e5])
def test_angles_of_the_frequencies(dev, base, layout):
    frequencies = rotary_frequencies(128, base)
    rotary = Rotary(frequencies, layout=layout, device=dev)
    g = torch.Generator(device=dev).manual_seed(1)
    q = torch.randn((len(POSITIONS), 4, 128), generator=g, device=dev).half()
    got = rotate(q, None, torch.tensor(POSITIONS, device=dev), rotary)[0].cpu().double()
    angle, off = (t[:, None] for t in angles(POSITIONS, frequencies))
    first, second = (slice(0, 64), slice(64, 128)) if layout == "half" else (slice(0, 128, 2), slice(1, 128, 2))
    x = q.cpu().double()
    a, b = x[..., first], x[..., second]
    cos, sin = angle.cos(), angle.sin()
    # A sine's series and roundings (2^-22), two products and a sum, the angle, and the output's rounding.
    reach = (a.abs() + b.abs()) * (2.0**-21 + off)
    for part, want in ((first, a * cos - b * sin), (second, a * sin + b * cos)):
        err = (got[..., part] - want).abs()
        assert bool((err <= reach + 2.0**-11 * (want.abs() + reach) + 2.0**-25).all())
