"""An attention block on NVFP4 weights over a key and value cache: the merged QKV
projection, packed attention and the output projection, as a server runs them.

    python examples/nvfp4_attention.py

Three prompts of different lengths go through the block at once, then each sequence
grows by one token at a time.  The last step is compared with the whole sequences
going through the block in one call.
"""

from __future__ import annotations

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from vflash_amd.attention import packed_attention  # noqa: E402
from vflash_amd.nvfp4_linear import NVFP4Execution, NVFP4Weight  # noqa: E402
from vflash_amd.prepare import quantize_nvfp4_weight  # noqa: E402


class Cache:
    """Keys and values of ``batch`` sequences, each with room for ``room`` tokens."""

    def __init__(self, batch, room, key_heads, dim, device, dtype=torch.bfloat16):
        self.k = torch.empty((batch * room, key_heads, dim), device=device, dtype=dtype)
        self.v = torch.empty_like(self.k)
        self.first = torch.arange(batch, device=device) * room  # each sequence's first row
        self.lengths = torch.zeros(batch, device=device, dtype=torch.int64)

    def append(self, k, v, offsets):
        """Adds the tokens ``offsets[b] .. offsets[b + 1]`` of ``k`` and ``v`` to sequence b."""
        token = torch.arange(k.shape[0], device=k.device)
        b = torch.searchsorted(offsets, token, right=True) - 1
        rows = self.first[b] + self.lengths[b] + token - offsets[b]
        self.k.index_copy_(0, rows, k)
        self.v.index_copy_(0, rows, v)
        self.lengths += offsets[1:] - offsets[:-1]


class AttentionBlock:
    """Grouped-head causal attention between two NVFP4 projections, weight-only."""

    def __init__(self, hidden, heads, key_heads, dim, device, seed=0):
        g = torch.Generator(device=device).manual_seed(seed)
        self.heads, self.key_heads, self.dim = heads, key_heads, dim
        self.execution = NVFP4Execution(activations="unquantized")

        def weight(n, k):
            w = torch.randn((n, k), generator=g, device=device) * k**-0.5
            return NVFP4Weight(*quantize_nvfp4_weight(w))

        self.qkv = weight((heads + 2 * key_heads) * dim, hidden)
        self.out = weight(hidden, heads * dim)

    @torch.no_grad()
    def __call__(self, x, offsets, cache):
        """``x`` [tokens, hidden], the new tokens of all sequences packed by ``offsets``."""
        merged = self.execution.linear(x, self.qkv).view(x.shape[0], -1, self.dim)
        q, k, v = merged.split((self.heads, self.key_heads, self.key_heads), dim=1)
        cache.append(k, v, offsets)
        attended = packed_attention(q, cache.k, cache.v, offsets, cache.first, k_lengths=cache.lengths, causal=True)
        return self.execution.linear(attended.flatten(1), self.out)


def packed(lengths, device):
    return torch.tensor([sum(lengths[:b]) for b in range(len(lengths) + 1)], dtype=torch.int64, device=device)


def run(device, prompts=(5, 130, 1), steps=8, hidden=512, heads=8, key_heads=2, dim=64):
    """The outputs of each sequence's last token, grown step by step and in one call."""
    block = AttentionBlock(hidden, heads, key_heads, dim, device)
    g = torch.Generator(device=device).manual_seed(1)
    tokens = [torch.randn((n + steps, hidden), generator=g, device=device).to(torch.bfloat16) for n in prompts]
    room = max(prompts) + steps

    cache = Cache(len(prompts), room, key_heads, dim, device)
    block(torch.cat([t[:n] for t, n in zip(tokens, prompts)]), packed(prompts, device), cache)
    one = packed([1] * len(prompts), device)
    for step in range(steps):
        grown = block(torch.stack([t[n + step] for t, n in zip(tokens, prompts)]), one, cache)

    whole = [n + steps for n in prompts]
    offsets = packed(whole, device)
    at_once = block(torch.cat(tokens), offsets, Cache(len(prompts), room, key_heads, dim, device))
    return grown, at_once[offsets[1:] - 1]


if __name__ == "__main__":
    grown, at_once = run(torch.device("cuda:0"))
    difference = ((grown - at_once).float().norm() / at_once.float().norm()).item()
    print(f"{grown.shape[0]} sequences grown token by token differ from one call by {difference:.1e} relative")
