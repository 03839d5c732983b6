"""The E4M3 codes of unrounded keys in a paged append, bit for bit."""

import pytest
import torch

from vflash_amd.paged import PagedCache, paged_append
from vflash_amd.rotary import Rotary, rotary_frequencies

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("heads,dim", [(8, 128), (3, 64), (5, 80), (7, 16)])
def test_codes_of_scaled_keys(dev, heads, dim, dtype):
    # At position 0 a rotation is its magnitude alone, one binary32 product, which the code is made of as it is.
    g = torch.Generator().manual_seed(dim)
    tokens, page = 2000, 64
    k = torch.randn((tokens, heads, dim), generator=g).to(dtype)
    k[5] = 0
    k[9, 1] *= 2.0**-80 if dtype == torch.bfloat16 else 2.0**-10  # one head of a wave far below the others
    table, n = torch.arange(32, device=dev)[None], torch.tensor([tokens], device=dev)
    offsets, at = torch.tensor([0, tokens], device=dev), torch.zeros(tokens, dtype=torch.int64, device=dev)
    for layout, magnitude in (("half", 1.2772588722239782), ("interleaved", 0.73), ("half", 1e-28)):
        cache = PagedCache.zeros(32, page, heads, dim, torch.float8_e4m3fn, dev)
        rotary = Rotary(rotary_frequencies(dim), layout=layout, magnitude=magnitude, device=dev)
        kd = k.to(dev)
        paged_append(cache, kd, kd, table, n, q_offsets=offsets, rotary=rotary, positions=at)
        x = k.float() * torch.tensor(magnitude, dtype=torch.float32)
        top = x.abs().amax(-1)
        scale = torch.where(top > 0, (top / 448.0).clamp_min(torch.finfo(torch.float32).tiny), torch.ones_like(top))
        codes = (x / scale[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
        got = cache.values[:, 0].permute(0, 2, 1, 3).reshape(32 * page, heads, dim)[:tokens].cpu()
        factors = cache.scales[:, 0].permute(0, 2, 1).reshape(32 * page, heads)[:tokens].cpu()
        assert torch.equal(factors, scale)
        assert torch.equal(got.view(torch.uint8), codes.view(torch.uint8))
