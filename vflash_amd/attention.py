"""Attention over packed sequences on MI355X, the operator between the merged QKV
projection and the attention output projection.

``packed_attention`` serves whole prompts packed one after another, pieces of prompts
appended to a cache, full (unmasked) attention, and single tokens over a cache, with
grouped heads.  The reference calls torch for it (src/vflash/native/h3_native_denoiser.py
applies attention between the two projections).  One HIP kernel family serves
every call (``vflash_packed_attention``); lengths stay on the device, so no call
synchronizes and a captured call replays with other lengths of the same total.
"""

from __future__ import annotations

import ctypes
import math

import torch

from vflash_amd import _lib, kernels


def packed_attention(q, k, v, q_offsets, k_offsets, *, k_lengths=None, causal=False, scale=None):
    """softmax(scale q k^T) v per sequence and head: ``[tokens, heads, dim]`` in q's type.

    ``q`` is bf16 or f16 ``[tokens, heads, dim]``, ``k`` and ``v`` are ``[keys, key_heads,
    dim]`` of the same type; ``heads`` is a multiple of ``key_heads`` and head ``h`` reads
    key head ``h // (heads // key_heads)``.  ``dim`` is a multiple of 8 up to 128.  Any
    strides are taken (slices of a merged projection, a transposed cache); a layout whose
    rows are not 16-byte runs is copied first.

    Sequence ``b`` has the queries ``q_offsets[b]`` to ``q_offsets[b + 1]`` and the keys
    ``k_offsets[b]`` to ``k_offsets[b + 1]`` (int64 device tensors of ``batch + 1``
    values).  With ``k_lengths`` (int64 ``[batch]``) it has ``k_lengths[b]`` keys from row
    ``k_offsets[b]`` (then ``[batch]`` too): a cache with room past each sequence, or one
    whose sequences share rows.  ``causal``: the queries are the sequence's last tokens,
    and query ``i`` of ``nq`` sees the keys ``j <= i + nk - nq``.  Rows that see no key, and
    rows outside every sequence, are zeros.  ``scale`` defaults to ``dim ** -0.5``.

    Offsets are read on the device, clamped to the operands.  A masked key has no effect,
    whatever it holds; infinities and NaN in its *value* may, as 0 times them is NaN, if it lies in its
    sequence.  No sum of finite values overflows; bf16 values below 2^-118 times the rows of ``k`` may
    lose bits to binary32's subnormals.  Inference only.
    """
    if isinstance(q, torch.Tensor) and q.is_cuda:
        # The whole call in native code; None sends any other layout, and every refusal, on from here.
        host = _lib.host()
        if host is not None:
            out = host.packed_attention(q, k, v, q_offsets, k_offsets, k_lengths, causal, scale)
            if out is not None:
                return out
    tensors = (q, k, v)
    if any(t.ndim != 3 for t in tensors):
        raise ValueError("packed attention takes [rows, heads, dim] queries, keys and values")
    if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("packed attention takes BF16 or F16 operands of one type")
    if k.shape != v.shape or k.shape[2] != q.shape[2]:
        raise ValueError("keys and values must have one shape and the queries' head dimension")
    heads, dim = q.shape[1:]
    key_heads = k.shape[1]
    if min(heads, key_heads) < 1 or heads % key_heads:
        raise ValueError("query heads must be a multiple of the key heads")
    if dim % 8 or not 8 <= dim <= 128:
        raise ValueError("the head dimension must be a multiple of 8 from 8 to 128")
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors) or kernels.has_tangent(*tensors):
        raise ValueError("packed attention is inference-only")
    batch = q_offsets.numel() - 1
    ends = batch if k_lengths is not None else batch + 1
    for name, t, length in (("q_offsets", q_offsets, batch + 1), ("k_offsets", k_offsets, ends),
                            ("k_lengths", k_lengths, batch)):
        if t is None:
            continue
        if t.dtype != torch.int64 or t.ndim != 1 or t.numel() != length or batch < 0 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int64 vector of the sequences")
    if scale is None:
        scale = 1.0 / math.sqrt(dim)
    elif not (ctypes.c_float(scale).value > 0.0 and scale <= 2.358e38):
        # times log2(e), in binary32
        raise ValueError("the scale must be positive and finite, and so must log2(e) times it")
    return kernels.packed_attention(q, k, v, q_offsets, k_offsets, k_lengths, bool(causal), scale)
