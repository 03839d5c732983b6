"""A serving step of many requests: an attention block on NVFP4 weights whose requests have adapters of their
own, rotary positions and a paged cache.

    python examples/serving_step.py

Requests of different lengths come in with their prompts, one in two pieces, then all grow by one token at a
time, in a batch padded to a fixed size as a captured step would be.  The last step is compared with the whole
sequences going through the block in one call, with the cache in bf16 and in E4M3.
"""

from __future__ import annotations

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from vflash_amd.adapters import add_request_adapters, stack_request_adapters  # noqa: E402
from vflash_amd.fused import LowRankResidual  # noqa: E402
from vflash_amd.nvfp4_linear import NVFP4Execution, NVFP4Weight  # noqa: E402
from vflash_amd.paged import PagedCache, paged_append, paged_attention  # noqa: E402
from vflash_amd.prepare import quantize_nvfp4_weight  # noqa: E402
from vflash_amd.rotary import Rotary, rotary_frequencies  # noqa: E402


class Pages:
    """The page table of ``batch`` sequences over one pool: pages are given out as sequences grow."""

    def __init__(self, batch, width, pages, page, device):
        self.page, self.device = page, device
        self.free = list(range(pages))
        self.own = [[] for _ in range(batch)]
        self.done = [0] * batch
        self.table = torch.zeros((batch, width), dtype=torch.int64, device=device)

    def grow(self, new):
        """Room for ``new[b]`` more tokens of sequence b; the lengths with them."""
        for b, n in enumerate(new):
            self.done[b] += n
            while len(self.own[b]) * self.page < self.done[b]:
                self.own[b].append(self.free.pop())
        for b, pages in enumerate(self.own):
            self.table[b, :len(pages)] = torch.tensor(pages, device=self.device)
        return torch.tensor(self.done, device=self.device)


class ServingBlock:
    """Grouped-head causal attention between two NVFP4 projections, weight-only; ``adapters`` adapters on Q, K and V."""

    def __init__(self, hidden, heads, key_heads, dim, adapters, device, seed=0):
        g = torch.Generator(device=device).manual_seed(seed)
        self.heads, self.key_heads, self.dim = heads, key_heads, dim
        self.execution = NVFP4Execution(activations="unquantized")

        def normal(*shape, std=1.0):
            return torch.randn(shape, generator=g, device=device) * std

        def weight(n, k):
            return NVFP4Weight(*quantize_nvfp4_weight(normal(n, k, std=k**-0.5)))

        self.qkv = weight((heads + 2 * key_heads) * dim, hidden)
        self.out = weight(hidden, heads * dim)
        self.rotary = Rotary(rotary_frequencies(dim), device=device)
        widths = (heads * dim, key_heads * dim, key_heads * dim)

        def residual(rank, n):
            return LowRankResidual(normal(rank, hidden, std=hidden**-0.5).to(torch.bfloat16),
                                   normal(n, rank, std=0.3 * rank**-0.5).to(torch.bfloat16), 0.75)

        self.adapters = stack_request_adapters([tuple(residual(4 + 6 * i, n) for n in widths) for i in range(adapters)],
                                               hidden, widths, device=device)

    @torch.no_grad()
    def __call__(self, x, adapter, cache, table, lengths, offsets=None):
        """``x`` [tokens, hidden]: the new tokens of all sequences packed by ``offsets``, or one of each; ``adapter``
        [tokens] their requests' adapters (-1: none)."""
        merged = self.execution.linear(x, self.qkv)
        merged = add_request_adapters(merged, x, self.adapters, adapter, inplace=True)
        q, k, v = merged.view(x.shape[0], -1, self.dim).split((self.heads, self.key_heads, self.key_heads), dim=1)
        q = paged_append(cache, k, v, table, lengths, q=q, q_offsets=offsets, rotary=self.rotary)
        attended = paged_attention(q, cache, table, lengths, q_offsets=offsets)
        return self.execution.linear(attended.flatten(1), self.out)


def packed(lengths, device):
    return torch.tensor([sum(lengths[:b]) for b in range(len(lengths) + 1)], dtype=torch.int64, device=device)


def run(device, store=torch.bfloat16, prompts=(5, 130, 1, 64), steps=8, hidden=512, heads=8, key_heads=2, dim=64, page=16):
    """The outputs of each sequence's last token, grown step by step and in one call."""
    block = ServingBlock(hidden, heads, key_heads, dim, 3, device)
    g = torch.Generator(device=device).manual_seed(1)
    tokens = [torch.randn((n + steps, hidden), generator=g, device=device).to(torch.bfloat16) for n in prompts]
    mine = [-1, 2, 0, 1][:len(prompts)]
    batch, whole = len(prompts), [n + steps for n in prompts]
    width = -(-max(whole) // page)

    def fresh(rows):
        return (PagedCache.zeros(rows * width, page, key_heads, dim, store, device),
                Pages(rows, width, rows * width, page, device))

    # The longest prompt in two pieces, the others with its first one.
    cache, pages = fresh(batch + 2)
    longest = max(range(batch), key=lambda b: prompts[b])
    done = [0] * batch
    for piece in ([n - n // 2 if b == longest else n for b, n in enumerate(prompts)],
                  [n // 2 if b == longest else 0 for b, n in enumerate(prompts)]):
        lengths = pages.grow([*piece, 0, 0])
        x = torch.cat([t[a:a + n] for t, a, n in zip(tokens, done, piece)])
        adapter = torch.tensor([a for a, n in zip(mine, piece) for _ in range(n)], device=device)
        block(x, adapter, cache, pages.table, lengths, packed([*piece, 0, 0], device))
        done = [a + n for a, n in zip(done, piece)]
    # Two rows of padding: sequences of no tokens.
    adapter = torch.tensor([*mine, -1, -1], device=device)
    rest = torch.zeros((2, hidden), device=device, dtype=torch.bfloat16)
    for step in range(steps):
        lengths = pages.grow([1] * batch + [0, 0])
        x = torch.cat((torch.stack([t[n + step] for t, n in zip(tokens, prompts)]), rest))
        grown = block(x, adapter, cache, pages.table, lengths)[:batch]

    cache, pages = fresh(batch)
    lengths, offsets = pages.grow(whole), packed(whole, device)
    adapter = torch.tensor([a for a, n in zip(mine, whole) for _ in range(n)], device=device)
    at_once = block(torch.cat(tokens), adapter, cache, pages.table, lengths, offsets)
    return grown, at_once[offsets[1:] - 1], block, tokens, mine


if __name__ == "__main__":
    for store in (torch.bfloat16, torch.float8_e4m3fn):
        grown, at_once, *_ = run(torch.device("cuda:0"), store)
        difference = ((grown - at_once).float().norm() / at_once.float().norm()).item()
        print(f"{store}: {grown.shape[0]} sequences grown token by token differ from one call by {difference:.1e} relative")
