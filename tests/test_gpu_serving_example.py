"""The example that runs the projections, the request adapters, rotary positions and the paged cache together."""

import importlib.util
import math
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
EXAMPLE = Path(__file__).resolve().parents[1] / "examples" / "serving_step.py"


def example():
    spec = importlib.util.spec_from_file_location("serving_step_example", EXAMPLE)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def dequantized(weight):
    """An NVFP4 weight in 64 bits, from its format."""
    codes = torch.stack((weight.packed & 15, weight.packed >> 4), -1).flatten(1).long()
    values = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=codes.device)
    w = values[codes & 7] * (1 - 2 * (codes >> 3))
    n, k = w.shape
    row, col = torch.arange(n, device=w.device)[:, None], torch.arange(k // 16, device=w.device)[None]
    at = row // 128 * (128 * (k // 16)) + col // 4 * 512 + row % 32 * 16 + row % 128 // 32 * 4 + col % 4
    scales = weight.scales.reshape(-1).view(torch.float8_e4m3fn).double()[at]
    return (w.view(n, k // 16, 16) * scales[..., None]).view(n, k) * weight.alpha.double()


def block_in_64_bits(block, x, adapter):
    """The block on one whole sequence, from the operators' definitions; the last token's output."""
    x = x.double()
    merged = x @ dequantized(block.qkv).T
    pack = block.adapters
    if adapter >= 0:
        width, first = pack.up.shape[2], 0
        for b, n in enumerate(pack.widths):
            low = x @ pack.down[adapter, b * width:(b + 1) * width].double().T
            merged[:, first:first + n] += pack.scaling[adapter, b].double() * low @ pack.up[adapter, first:first + n].double().T
            first += n
    h, g, d = block.heads, block.key_heads, block.dim
    q, k, v = merged.view(len(x), -1, d).split((h, g, g), 1)
    phases = block.rotary.phases.double() * 2.0**-64 * 2 * math.pi
    turn = torch.polar(torch.ones_like(phases).expand(len(x), -1), torch.arange(len(x), device=x.device)[:, None] * phases)[:, None]

    def rotated(t):
        z = torch.complex(t[..., :d // 2], t[..., d // 2:]) * turn
        return torch.cat((z.real, z.imag), -1)

    q, k = rotated(q)[-1], rotated(k)
    p = torch.softmax(torch.einsum("hd,nhd->hn", q, k.repeat_interleave(h // g, 1)) / math.sqrt(d), -1)
    return torch.einsum("hn,nhd->hd", p, v.repeat_interleave(h // g, 1)).flatten() @ dequantized(block.out).T


@pytest.mark.parametrize("store", [torch.bfloat16, torch.float8_e4m3fn], ids=["bf16", "e4m3"])
def test_growing_sequences_agree_with_whole_ones(dev, store):
    grown, whole, block, tokens, mine = example().run(dev, store)
    assert grown.shape == whole.shape == (4, 512) and bool(torch.isfinite(grown).all())
    want = torch.stack([block_in_64_bits(block, x, a) for x, a in zip(tokens, mine)])
    # Rounded to bf16, by half a step (2^-8 of the value) at most: the projection, the sum with the adapter, q and k after
    # their rotation, the weights, the attention's output and the result; q and k move a score of size s by 2 * 3
    # of these halves of it, and scores are below 4 here.  E4M3 moves keys and values by 2^-4 of themselves at most.
    # Errors of single values add up as norms, and are a third of their bound in the mean.
    half = 2.0**-8
    bound = (6 + 4 * 6) * half / 3 + (0 if store == torch.bfloat16 else (1 + 4) * 2.0**-4 / 3)
    for got in (grown, whole):
        assert (got.double() - want).norm() <= bound * want.norm()
    # The two differ where a sum's order moves a rounding by a whole step, of a code with E4M3.
    assert (grown - whole).double().norm() <= (4 * 2.0**-7 if store == torch.bfloat16 else 2.0**-4) * whole.double().norm()


def test_requests_with_adapters_differ(dev):
    # The adapters reach the output, and only their own requests'.
    module = example()
    block = module.ServingBlock(512, 8, 2, 64, 2, dev)
    x = torch.randn((3, 512), device=dev).to(torch.bfloat16)
    n, table = torch.ones(3, dtype=torch.int64, device=dev), torch.arange(3, device=dev)[:, None].contiguous()

    def step(adapter):
        cache = module.PagedCache.zeros(3, 16, 2, 64, device=dev)
        return block(x, torch.tensor(adapter, device=dev), cache, table, n)

    none, some = step([-1, -1, -1]), step([-1, 1, 0])
    assert torch.equal(none[0], some[0]) and not torch.equal(none[1], some[1]) and not torch.equal(none[2], some[2])
