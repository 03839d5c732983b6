"""A paged cache of keys and values on MI355X, the append of new tokens to it and the attention
that reads it.

``PagedCache`` holds pages in the operands' 16-bit type or in E4M3 with a scale for each row, as
the row-FP8 linears quantize.  ``paged_append`` stores the keys and values of a step and
rotates queries and keys on the way, in one launch; ``paged_attention`` attends with them.  Both
take the same page table, lengths and offsets, all on the device: no call synchronizes,
and a captured step replays with other lengths and pages.  The contiguous form is
``attention.packed_attention``.
"""

from __future__ import annotations

import ctypes
import math

import torch

from vflash_amd import _lib, kernels
from vflash_amd.rotary import Rotary, check_heads, check_positions, check_rotary


class PagedCache:
    """``values`` is ``[pages, 2, key_heads, page, dim]``, contiguous: each page holds, head by head, the
    keys of ``page`` tokens and then their values, so that a head's keys of a page are one run of
    memory.  bf16 or f16, or ``float8_e4m3fn`` with ``scales``, fp32 ``[pages, 2, key_heads, page]``.
    ``page`` is a power of two from 16 to 4096; ``dim`` a multiple of 8 (of 16 in E4M3) up to 128.
    """

    __slots__ = ("values", "scales")

    def __init__(self, values, scales=None):
        if values.ndim != 5 or values.shape[1] != 2 or not values.is_contiguous():
            raise ValueError("a paged cache is a contiguous [pages, 2, key_heads, page, dim] tensor")
        page, dim = values.shape[3:]
        if not 16 <= page <= 4096 or page & (page - 1):
            raise ValueError("a page holds a power of two of tokens, from 16 to 4096")
        codes = values.dtype == torch.float8_e4m3fn
        if not codes and values.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("a paged cache is BF16, F16 or E4M3")
        if dim % (16 if codes else 8) or not 8 <= dim <= 128:
            raise ValueError("the head dimension must be a multiple of 8 (16 in E4M3) up to 128")
        if not 1 <= values.shape[2] <= 4096:
            raise ValueError("a paged cache has 1 to 4096 key heads")
        if codes != (scales is not None):
            raise ValueError("E4M3 pages, and they alone, come with scales")
        if codes and (scales.dtype != torch.float32 or scales.shape != values.shape[:4] or not scales.is_contiguous()
                      or scales.device != values.device):
            raise ValueError("scales must be a contiguous fp32 [pages, 2, key_heads, page] tensor beside the pages")
        if any(t is not None and (t.requires_grad or t.is_neg() or t.data_ptr() % 16) for t in (values, scales)):
            raise ValueError("a paged cache is plain memory, 16-byte aligned, without gradients")
        object.__setattr__(self, "values", values)
        object.__setattr__(self, "scales", scales)

    def __setattr__(self, name, value):
        raise AttributeError("a paged cache keeps the tensors that it was made of")

    def __reduce__(self):
        # As bytes where they are codes: pickle has no name for torch's storage of these.
        values = self.values if self.scales is None else self.values.view(torch.uint8)
        return _cache_of, (type(self), values, self.scales)

    @classmethod
    def zeros(cls, pages, page, key_heads, dim, dtype=torch.bfloat16, device="cuda"):
        """An empty cache."""
        values = torch.zeros((pages, 2, key_heads, page, dim), dtype=dtype, device=device)
        scales = None
        if dtype == torch.float8_e4m3fn:
            scales = torch.ones((pages, 2, key_heads, page), dtype=torch.float32, device=device)
        return cls(values, scales)


def _cache_of(cls, values, scales):
    """What ``copy`` and ``pickle`` make of another's tensors, which are checked as those were."""
    return cls(values if scales is None else values.view(torch.float8_e4m3fn), scales)


def _plain(t):
    return t.is_contiguous() and not t.is_neg()


def _check_sequences(tokens, table, lengths, q_offsets):
    if table.dtype != torch.int64 or table.ndim != 2 or table.shape[1] < 1 or not _plain(table):
        raise ValueError("the page table must be a contiguous int64 [batch, pages] tensor")
    batch = table.shape[0]
    for name, t, length in (("lengths", lengths, batch), ("q_offsets", q_offsets, batch + 1)):
        if t is not None and (t.dtype != torch.int64 or t.ndim != 1 or t.numel() != length or not _plain(t)):
            raise ValueError(f"{name} must be a contiguous int64 vector of the sequences")
    if q_offsets is None and tokens != batch:
        raise ValueError("without q_offsets every sequence has one token")


def _check_store(cache, q, key_heads):
    if not isinstance(cache, PagedCache):
        raise ValueError("paged attention takes a PagedCache")
    if cache.values.shape[2] != key_heads or cache.values.shape[4] != q.shape[2]:
        raise ValueError("the paged cache has other heads")
    if cache.scales is None and cache.values.dtype != q.dtype:
        raise ValueError("the paged cache has another type")


def paged_append(cache: PagedCache, k, v, table, lengths, *, q=None, q_offsets=None, rotary: Rotary | None = None,
                 positions=None):
    """Stores the keys and values of new tokens; returns ``q`` rotated (None without ``q``).

    ``k`` and ``v`` are bf16 or f16 ``[tokens, key_heads, dim]``, ``q`` ``[tokens, heads, dim]``, of one
    type (the cache's, unless that is E4M3), with any strides.  Sequence ``b``'s new tokens are
    ``q_offsets[b]`` to ``q_offsets[b + 1]`` (int64 ``[batch + 1]``; None: one token a sequence), and
    ``lengths[b]`` (int64 ``[batch]``) counts its tokens with the new ones: token ``i`` of ``n`` new
    ones is the sequence's token ``lengths[b] - n + i``, kept in slot ``i % page`` of page
    ``table[b, i // page]`` (int64 ``[batch, width]``).

    ``rotary`` rotates ``k`` and ``q`` to the tokens' places in their sequences, or to ``positions`` (int64
    ``[tokens]`` or ``[tokens, axes]``) where a model counts otherwise.  E4M3 rows are quantized from the
    unrounded rotated values.

    A token without a place (outside the offsets, in a sequence of length 0, past the table or on a page
    that does not exist) is not stored, and its rows of ``q`` come back as zeros: a batch
    padded with sequences of length 0 leaves the cache alone.  Inference only.
    """
    if (isinstance(k, torch.Tensor) and k.is_cuda and isinstance(cache, PagedCache)
            and (rotary is None or isinstance(rotary, Rotary))):
        # The whole call in native code; None sends any other layout, and every refusal, on from here.
        host = _lib.host()
        if host is not None:
            r = (None, None, 1, False, 1.0) if rotary is None else (
                rotary.phases, rotary.axis, rotary.axes, rotary.interleaved, rotary.magnitude)
            out = host.paged_append(q, k, v, cache.values, cache.scales, table, lengths, q_offsets, positions, *r)
            if out is not None:
                return out if q is not None else None
    tensors = [k, v] if q is None else [k, v, q]
    check_heads("the paged append", tensors, 128)
    if v.shape != k.shape or (q is not None and q.shape[0] != k.shape[0]):
        raise ValueError("the paged append takes keys, values and queries of the same tokens")
    _check_store(cache, k, k.shape[1])
    _check_sequences(k.shape[0], table, lengths, q_offsets)
    if rotary is None:
        if q is not None or positions is not None:
            raise ValueError("queries and positions come with rotary positions")
    else:
        check_rotary(rotary, k.shape[2])
        if positions is not None:
            check_positions(positions, k.shape[0], rotary)
        elif rotary.axes > 1:
            raise ValueError("pairs that follow several axes need positions")
    return kernels.paged_append(cache, q, k, v, table, lengths, q_offsets, rotary, positions)


def paged_attention(q, cache: PagedCache, table, lengths, *, q_offsets=None, scale=None):
    """softmax(scale q k^T) v of new tokens over the paged cache that holds them: ``[tokens, heads, dim]``.

    The cache, ``table``, ``lengths`` and ``q_offsets`` are those of ``paged_append`` (which comes first);
    ``heads`` is a multiple of the cache's key heads, and head ``h`` reads key head
    ``h // (heads // key_heads)``.  One token a sequence without ``q_offsets``, else any number (drafted tokens, a
    prompt or its next piece): token ``i`` of ``n`` sees the sequence's first ``lengths[b] - n + i + 1`` tokens.  Rows that
    see none, and rows outside every sequence, are zeros.  ``scale`` defaults to ``dim ** -0.5``.

    Single tokens, drafts and short pieces run in tiles of 16 rows (token and head), prompts and longer pieces in
    tiles of 128, as in ``packed_attention``.  Softmax and sums are binary32; weights are rounded to the operands'
    type; with an E4M3 cache to bf16 after the values' scales, for f16 queries to two bf16.  As there, infinities and
    NaN in the values of a sequence can reach its masked queries as NaN.  Inference only.

    The lengths stay on the device, so the launch is chosen by the table's room (its width times the page) in their
    place.  Pass a table as wide as the longest sequence needs where that is known (``table[:, :n].contiguous()``): 77 keys
    take 7.2 us in a room of 77 and 10.6 in one of 2048 or more, 128 single tokens over 200 keys 22 and 35, five drafts
    after 500 11.5 and, in a room of 131072, 20.8.  A captured step keeps the room that it was captured with.
    """
    if isinstance(q, torch.Tensor) and q.is_cuda and isinstance(cache, PagedCache):
        host = _lib.host()
        if host is not None:
            out = host.paged_attention(q, cache.values, cache.scales, table, lengths, q_offsets, scale)
            if out is not None:
                return out
    check_heads("paged attention", [q], 128)
    if not isinstance(cache, PagedCache):
        raise ValueError("paged attention takes a PagedCache")
    key_heads = cache.values.shape[2]
    _check_store(cache, q, key_heads)
    if q.shape[1] % key_heads:
        raise ValueError("query heads must be a multiple of the key heads")
    _check_sequences(q.shape[0], table, lengths, q_offsets)
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[2])
    elif not (ctypes.c_float(scale).value > 0.0 and scale <= 2.358e38):
        # times log2(e), in binary32
        raise ValueError("the scale must be positive and finite, and so must log2(e) times it")
    return kernels.paged_attention(q, cache, table, lengths, q_offsets, scale)
