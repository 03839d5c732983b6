"""The low-rank adapters of many requests beside one projection on MI355X.

``fused.fp8_linear_lora`` and the other adapter epilogues serve one adapter (or one for each merged
branch) a call; in a batch of requests each row has its own.  ``RequestAdapters`` keeps the adapters of a
projection side by side and ``add_request_adapters`` adds, to each row of its output, the
delta of the row's adapter.  It stands beside any projection of the package (W8A8, NVFP4 in its
three forms) on the projection's 16-bit input and output.
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass, field

import torch

from vflash_amd import _lib, kernels
from vflash_amd.fused import LowRankResidual

MAX_BRANCHES = 3
MAX_ADAPTERS = 8191


@dataclass(frozen=True, eq=False)
class RequestAdapters:
    """Adapters of one projection of ``k`` inputs, or of up to three merged ones (Q, K and V) of
    ``widths`` outputs each.

    ``down`` is ``[adapters, branches * width, k]`` and ``up`` ``[adapters, sum(widths), width]``, bf16 or f16, where
    ``width`` (a multiple of 16 up to 128) holds the largest rank; rows of ``down`` and columns of ``up`` at and past
    an adapter's rank are zeros.  ``scaling`` is fp32 ``[adapters, branches]``, ``ranks`` int32
    ``[adapters]`` (the largest of its branches).  ``stack_request_adapters`` lays them out; one slot's tensors can be
    overwritten in place when another adapter takes it.
    """

    down: torch.Tensor
    up: torch.Tensor
    scaling: torch.Tensor
    ranks: torch.Tensor
    widths: tuple
    c_widths: object = field(init=False, repr=False)

    def __post_init__(self):
        down, up, widths = self.down, self.up, tuple(int(w) for w in self.widths)
        if not 1 <= len(widths) <= MAX_BRANCHES or any(w < 8 or w % 8 or w >= 1 << 21 for w in widths):
            raise ValueError("request adapters take one to three branches, whose widths are multiples of 8")
        if down.dtype not in (torch.bfloat16, torch.float16) or up.dtype != down.dtype:
            raise ValueError("request adapters are BF16 or F16 matrices of one type")
        if down.ndim != 3 or up.ndim != 3 or not 1 <= down.shape[0] <= MAX_ADAPTERS or up.shape[0] != down.shape[0]:
            raise ValueError(f"request adapters are stacks of 1 to {MAX_ADAPTERS}")
        width = up.shape[2]
        if width % 16 or not 16 <= width <= kernels.LORA_MAX_RANK or down.shape[1] != len(widths) * width:
            raise ValueError("request adapters hold ranks padded to a multiple of 16 up to 128")
        if up.shape[1] != sum(widths) or down.shape[2] < 8 or down.shape[2] % 8:
            raise ValueError("request adapters do not match the projection")
        if self.scaling.shape != (down.shape[0], len(widths)) or self.scaling.dtype != torch.float32:
            raise ValueError("request adapters take one fp32 scaling for each adapter and branch")
        if self.ranks.shape != (down.shape[0],) or self.ranks.dtype != torch.int32:
            raise ValueError("request adapters take one int32 rank for each adapter")
        for t in (down, up, self.scaling, self.ranks):
            if t.device != down.device or not t.is_contiguous() or t.is_neg() or t.requires_grad or t.data_ptr() % 16:
                raise ValueError("request adapters are contiguous tensors of one device, without gradients")
        object.__setattr__(self, "widths", widths)
        object.__setattr__(self, "c_widths", (ctypes.c_int64 * len(widths))(*widths))

    def __reduce__(self):  # copy and pickle: c_widths is made again, and the tensors are checked as these were
        return type(self), (self.down, self.up, self.scaling, self.ranks, self.widths)


def stack_request_adapters(adapters, k: int, widths, *, dtype=torch.bfloat16, device="cuda") -> RequestAdapters:
    """``RequestAdapters`` of a list of adapters, each a ``LowRankResidual`` or, for merged branches, a tuple with
    one or None for each.  Done once when adapters are loaded."""
    widths = tuple(widths)
    packs = [a if isinstance(a, (tuple, list)) else (a,) for a in adapters]
    if not packs:
        raise ValueError("request adapters are a stack of one at least")
    for pack in packs:
        if len(pack) != len(widths):
            raise ValueError("request adapters take one adapter, or None, for each branch")
        for r, n in zip(pack, widths):
            if r is None:
                continue
            if not isinstance(r, LowRankResidual):
                raise ValueError("adapters must be LowRankResidual weights")
            if r.down.ndim != 2 or r.up.ndim != 2 or r.down.shape[0] < 1 or r.up.shape[1] != r.down.shape[0]:
                raise ValueError("Adapter projection requires compatible nonempty A/B matrices")
            if r.down.shape[1] != k or r.up.shape[0] != n:
                raise ValueError("Adapter projection does not match the target model")
            if r.down.shape[0] > kernels.LORA_MAX_RANK:
                raise ValueError(f"request adapters take ranks up to {kernels.LORA_MAX_RANK}")
            if not math.isfinite(r.scaling) or isinstance(r.scaling, bool):
                raise ValueError("Adapter scale must be finite")
    ranks = [max((r.down.shape[0] for r in pack if r is not None), default=0) for pack in packs]
    width = max(16, -(-max(ranks) // 16) * 16)
    down = torch.zeros((len(packs), len(widths) * width, k), dtype=dtype, device=device)
    up = torch.zeros((len(packs), sum(widths), width), dtype=dtype, device=device)
    scaling = torch.zeros((len(packs), len(widths)), dtype=torch.float32, device=device)
    for i, pack in enumerate(packs):
        first = 0
        for b, (r, n) in enumerate(zip(pack, widths)):
            if r is not None:
                rank = r.down.shape[0]
                down[i, b * width:b * width + rank] = r.down
                up[i, first:first + n, :rank] = r.up
                scaling[i, b] = r.scaling
            first += n
    return RequestAdapters(down, up, scaling, torch.tensor(ranks, dtype=torch.int32, device=device), widths)


def add_request_adapters(base, x, adapters: RequestAdapters, index, *, inplace: bool = False):
    """``base[m] + scaling (x[m] down^T) up^T`` of each row's adapter ``index[m]``.

    ``x`` is the projection's input ``[.., k]`` and ``base`` its output ``[.., sum(widths)]``, bf16 or f16 as the adapters
    are; ``index`` is int64 with one value for each row, read on the device: a captured call replays
    with other adapters.  A row whose index is outside the stack (-1) has no adapter and keeps its value.  Rows
    may come in any order; each adapter in use is read about once.  ``inplace`` writes to ``base``.

    Sums are binary32 and the result is rounded once (the one-adapter epilogues round each step, as the
    reference's hook does).  Infinities and NaN of a row of ``x`` reach all branches of its adapter.  Inference only.
    """
    if isinstance(base, torch.Tensor) and base.is_cuda and isinstance(adapters, RequestAdapters):
        # The whole call in native code; None sends any other layout, and every refusal, on from here.
        host = _lib.host()
        if host is not None:
            out = host.request_adapters(base, x, adapters.down, adapters.up, adapters.scaling, adapters.ranks,
                                        adapters.widths, index, inplace)
            if out is not None:
                return out
    if not isinstance(adapters, RequestAdapters):
        raise ValueError("many adapters come as RequestAdapters")
    n, k = adapters.up.shape[1], adapters.down.shape[2]
    if x.ndim < 1 or base.ndim < 1 or x.shape[-1] != k or base.shape[-1] != n or x.shape[:-1] != base.shape[:-1]:
        raise ValueError("Adapter projection does not match the target model")
    if x.dtype != adapters.down.dtype or base.dtype != x.dtype:
        raise ValueError("request adapters take inputs and outputs of their own type")
    if torch.is_grad_enabled() and (x.requires_grad or base.requires_grad) or kernels.has_tangent(x, base):
        raise ValueError("request adapters are inference-only")
    if index.dtype != torch.int64 or index.numel() != base.shape[:-1].numel() or not index.is_contiguous():
        raise ValueError("adapter indices must be a contiguous int64 tensor with one value for each row")
    return kernels.request_adapters(base, x, adapters, index, inplace)
