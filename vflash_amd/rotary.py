"""Rotary positions on MI355X: the query and key heads between the merged QKV projection
and attention.

``Rotary`` holds what a model keeps (its frequencies, the layout of the pairs, the axes that
they follow), ``rotate`` applies it to queries and keys in one launch, and
``paged.paged_append`` does so on the way into a paged cache.  The reference rotates split
halves by a table of cosines (src/vflash/native/h3_fused_ops.py:428-507); here the
angles are formed in the kernel from integers, and no table is read.  An angle is off by
``2 ** -33 + abs(position) * 2 ** -65`` of a turn at most: 1.5e-9 rad up to position ``2 ** 32``.
"""

from __future__ import annotations

import math
from fractions import Fraction

import torch

from vflash_amd import _lib, kernels

# 2^200 / (2 pi)
_PER_TURN = round(2**200 / Fraction("6.2831853071795864769252867665590057683943387987502116419498891846156328125724"))
LAYOUTS = ("half", "interleaved")


def rotary_frequencies(dim: int, base: float = 10000.0, *, scaling: str | None = None, factor: float = 1.0,
                       context: int | None = None, low: float = 1.0, high: float = 32.0) -> list[float]:
    """Radians a position of the ``dim / 2`` pairs: ``base ** (-2 i / dim)``, for contexts longer than
    the model was trained on changed by ``scaling``:

    * ``"linear"``: all divided by ``factor``;
    * ``"base"``: ``base`` times ``factor ** (dim / (dim - 2))``, so that the slowest pair is divided by
      ``factor`` and the fastest stays;
    * ``"parts"``: pairs that turn at most ``low`` times in ``context`` positions are divided by
      ``factor``, those that turn ``high`` times or more stay, those between are interpolated in
      their number of turns.
    """
    if dim < 2 or dim % 2:
        raise ValueError("rotary positions take an even number of dimensions")
    if not (math.isfinite(base) and base > 0) or not (math.isfinite(factor) and factor > 0):
        raise ValueError("the rotary base and factor must be positive and finite")
    if scaling not in (None, "linear", "base", "parts"):
        raise ValueError("unknown rotary scaling")
    if scaling == "base":
        if dim < 4:
            raise ValueError("scaling the base takes at least two pairs")
        base *= factor ** (dim / (dim - 2))
    f = [base ** (-2.0 * i / dim) for i in range(dim // 2)]
    if scaling == "linear":
        return [x / factor for x in f]
    if scaling == "parts":
        if context is None or context < 1 or not high > low:
            raise ValueError("scaling by parts takes the trained context and low < high")
        keep = [min(1.0, max(0.0, (context * x / (2 * math.pi) - low) / (high - low))) for x in f]
        return [x * (g + (1.0 - g) / factor) for x, g in zip(f, keep)]
    return f


def _phase(frequency: float) -> int:
    """Turns a position in 2^-64, modulo one turn, as a signed 64-bit word: to nearest, in integers, so that
    ``position`` of them are ``abs(position) * 2 ** -65`` of a turn off at most."""
    n, d = frequency.as_integer_ratio()  # d is a power of two
    shift = 135 + d.bit_length()  # 200 - 64 + log2(d)
    turns = (n * _PER_TURN + (1 << (shift - 1)) >> shift) + 2**63
    return turns % 2**64 - 2**63


class Rotary:
    """Rotary positions of heads of at least ``2 * len(frequencies)`` dimensions.

    ``frequencies`` are radians a position, one for each pair.  Pair ``i`` is the elements
    ``i`` and ``i + pairs`` of a head (``"half"``) or ``2 i`` and ``2 i + 1`` (``"interleaved"``);
    elements past the pairs are left as they are.  ``axes`` gives, for each pair, which of a
    token's positions it follows (a video's frame, row and column); without it every
    pair follows the one position.  ``magnitude`` multiplies the rotated elements, as some
    scalings for long contexts ask.
    """

    __slots__ = ("phases", "axis", "axes", "pairs", "interleaved", "magnitude")

    def __init__(self, frequencies, *, layout: str = "half", axes=None, magnitude: float = 1.0, device="cuda"):
        frequencies = [float(f) for f in frequencies]
        if layout not in LAYOUTS:
            raise ValueError(f"the rotary layout is one of {LAYOUTS}")
        if not frequencies or not all(math.isfinite(f) for f in frequencies):
            raise ValueError("rotary positions take one finite frequency for each pair")
        # within binary32, as the kernel multiplies
        if not abs(magnitude) <= 3.39e38:
            raise ValueError("the rotary magnitude must be finite")
        axis, count = None, 1
        if axes is not None:
            axes = [int(a) for a in axes]
            if len(axes) != len(frequencies) or min(axes) < 0 or max(axes) > 63:
                raise ValueError("rotary axes are one of 0 to 63 for each pair")
            count = max(axes) + 1
            if count > 1:
                axis = torch.tensor(axes, dtype=torch.int64, device=device)
        phases = torch.tensor([_phase(f) for f in frequencies], dtype=torch.int64, device=device)
        self._keep(phases, axis, count, layout == "interleaved", float(magnitude))

    def _keep(self, phases, axis, axes, interleaved, magnitude):
        for name, value in (("phases", phases), ("pairs", phases.numel()), ("interleaved", interleaved),
                            ("magnitude", magnitude), ("axis", axis), ("axes", axes)):
            object.__setattr__(self, name, value)

    def __setattr__(self, name, value):
        raise AttributeError("rotary positions keep what they were made of")

    def __reduce__(self):
        return _rotary_of, (type(self), self.phases, self.axis, self.axes, self.interleaved, self.magnitude)


def _rotary_of(cls, phases, axis, axes, interleaved, magnitude):
    """What ``copy`` and ``pickle`` make of the parts that another was kept in."""
    for t in (phases, axis):
        if t is not None and (t.dtype != torch.int64 or t.shape != (max(phases.numel(), 1),) or not t.is_contiguous()
                              or t.device != phases.device):
            raise ValueError("rotary phases and axes are int64 vectors of one length")
    if not 1 <= axes <= 64 or (axes == 1) != (axis is None) or not abs(magnitude) <= 3.39e38:
        raise ValueError("rotary positions of unknown parts")
    rotary = cls.__new__(cls)
    rotary._keep(phases, axis, int(axes), bool(interleaved), float(magnitude))
    return rotary


def rotate(q, k, positions, rotary: Rotary):
    """``q`` and ``k`` rotated to ``positions``: new contiguous tensors of their types; ``k`` may be None.

    ``q`` is bf16 or f16 ``[tokens, heads, dim]`` and ``k`` ``[tokens, key_heads, dim]`` of the same
    type; ``dim`` is a multiple of 8 up to 256 that holds the pairs.  Any strides are taken
    (slices of a merged projection); a layout whose rows are not 16-byte runs is copied
    first.  ``positions`` is int64 ``[tokens]``, or ``[tokens, axes]`` where the pairs follow
    several, of any values (a negative position turns back); angles lose bits past ``2 ** 32``, as above.

    ``(a, b)`` becomes ``magnitude (a cos - b sin, a sin + b cos)`` in binary32, rounded once.  Inference only.
    """
    if isinstance(q, torch.Tensor) and q.is_cuda and isinstance(rotary, Rotary):
        # The whole call in native code; None sends any other layout, and every refusal, on from here.
        host = _lib.host()
        if host is not None:
            out = host.rotate(q, k, positions, rotary.phases, rotary.axis, rotary.axes, rotary.interleaved, rotary.magnitude)
            if out is not None:
                return out
    tensors = [q] if k is None else [q, k]
    check_heads("rotary positions", tensors, 256)
    if k is not None and k.shape[0] != q.shape[0]:
        raise ValueError("rotary positions take queries and keys of the same tokens")
    check_rotary(rotary, q.shape[2])
    check_positions(positions, q.shape[0], rotary)
    return kernels.rotate(q, k, positions, rotary)


def check_heads(what, tensors, most):
    """bf16 or f16 ``[tokens, heads, dim]`` of one type and dim, without gradients."""
    for t in tensors:
        if t.ndim != 3 or t.shape[1] < 1:
            raise ValueError(f"{what}: [tokens, heads, dim] tensors")
        if t.dtype not in (torch.bfloat16, torch.float16) or t.dtype != tensors[0].dtype:
            raise ValueError(f"{what}: BF16 or F16 operands of one type")
        if t.shape[2] != tensors[0].shape[2]:
            raise ValueError(f"{what}: operands of one head dimension")
    dim = tensors[0].shape[2]
    if dim % 8 or not 8 <= dim <= most:
        raise ValueError(f"{what}: the head dimension must be a multiple of 8 from 8 to {most}")
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors) or kernels.has_tangent(*tensors):
        raise ValueError(f"{what}: inference-only")


def check_rotary(rotary, dim):
    if not isinstance(rotary, Rotary):
        raise ValueError("rotary positions take a Rotary")
    if 2 * rotary.pairs > dim:
        raise ValueError("the heads are smaller than the rotary pairs")


def check_positions(positions, tokens, rotary):
    shapes = [(tokens, rotary.axes)] + ([(tokens,)] if rotary.axes == 1 else [])
    if positions.dtype != torch.int64 or tuple(positions.shape) not in shapes:
        raise ValueError("rotary positions must be int64, one of each axis for each token")
