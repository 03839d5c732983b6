"""The paged cache on the GPU: what the append stores, and attention over it against its definition in 64 bits."""

import random

import pytest
import torch

from tests.attention_reference import check, packed_attention
from tests.test_gpu_rotary import turned
from vflash_amd import _lib, attention, kernels
from vflash_amd.paged import PagedCache, paged_append, paged_attention
from vflash_amd.rotary import Rotary, rotary_frequencies

pytestmark = pytest.mark.gpu
BF16, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def offsets(lengths, dev):
    return torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int64, device=dev)


def make(dev, *shape, dtype=BF16, seed=0, std=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=dev) * std).to(dtype)


def pool(dev, lengths, page, kv, dim, dtype, seed=0, spare=2, width=None):
    """A cache with random contents, and a table of pages in random order (-1 past a sequence's own)."""
    need = [-(-max(n, 0) // page) for n in lengths]
    pages = sum(need) + spare
    order = list(range(pages))
    random.Random(seed).shuffle(order)
    width = width or max(max(need, default=0), 1)
    table = [[-1] * width for _ in lengths]
    for row, n in zip(table, need):
        row[:n] = [order.pop() for _ in range(n)]
    table = torch.tensor(table, dtype=torch.int64, device=dev).view(len(lengths), width)
    values = make(dev, pages, 2, kv, page, dim, dtype=torch.float32, seed=seed)
    if dtype == E4M3:
        values *= torch.rand(pages, 2, kv, page, 1, device=dev) * 3 + 0.1
        scales = values.abs().amax(-1) / 448
        return PagedCache((values / scales[..., None]).clamp(-448, 448).to(E4M3), scales), table
    return PagedCache(values.to(dtype)), table


def stored(cache):
    """What the cache holds, in 64 bits."""
    values = cache.values.double()
    return values if cache.scales is None else values * cache.scales.double().unsqueeze(-1)


def rows_of(cache, table, lengths):
    """Keys and values one sequence after another, [keys, heads, dim], on the CPU in 64 bits."""
    all_values, page = stored(cache).cpu(), cache.values.shape[3]
    parts = []
    for row, n in zip(table.tolist(), lengths):
        at = [all_values[row[i // page], :, :, i % page] for i in range(n)]
        parts += at
    empty = torch.zeros((0, *all_values.shape[1:3], all_values.shape[4]), dtype=torch.float64)
    rows = torch.stack(parts) if parts else empty
    return rows[:, 0], rows[:, 1]


def attended(cache, q, table, lengths, q_offsets, got, scale=None):
    k, v = rows_of(cache, table, lengths)
    qo = torch.arange(len(lengths) + 1) if q_offsets is None else q_offsets
    ko = offsets(lengths, "cpu")
    if cache.scales is None:
        check(got, q, k.to(q.dtype), v.to(q.dtype), qo, ko, causal=True, scale=scale)
        return
    # E4M3: weights round to bf16, for f16 to two of it (2^-17, inside binary16's half step), and normalise unrounded; a
    # factor's product is one binary32 rounding more in a score and in a weight.
    want, bound = packed_attention(q, k, v, qo, ko, causal=True, scale=scale)
    got = got.cpu().double()
    assert bool(torch.isfinite(got).all())
    worst = ((got - want).abs() - bound).max().item()
    assert worst <= 0, f"{worst} past the bound"


# ---------------------------------------------------------------------------
APPENDS = [([1], [1]), ([1], [77]), ([1, 1, 1], [5, 16, 17]), ([5], [5]), ([0, 3, 40], [7, 3, 100]), ([33, 0, 1], [33, 0, 64]),
           ([70] * 5, [70, 71, 90, 200, 100])]


@pytest.mark.parametrize("dtype,store", [(BF16, BF16), (F16, F16), (BF16, E4M3), (F16, E4M3)])
@pytest.mark.parametrize("heads,kv,dim,page", [(8, 2, 128, 16), (4, 4, 64, 64), (6, 1, 96, 32), (10, 5, 80, 16), (3, 3, 16, 128)])
@pytest.mark.parametrize("new,lengths", APPENDS, ids=lambda v: "-".join(map(str, v)))
def test_append(dev, new, lengths, heads, kv, dim, page, dtype, store):
    cache, table = pool(dev, lengths, page, kv, dim, store)
    tokens = sum(new)
    q, k, v = make(dev, tokens, heads + 2 * kv, dim, dtype=dtype, seed=3).split((heads, kv, kv), 1)
    before = cache.values.view(torch.uint8).clone()
    scales = None if cache.scales is None else cache.scales.clone()
    rotary = Rotary(rotary_frequencies(dim), layout="half" if page == 16 else "interleaved", device=dev)
    qo = None if new == [1] * len(new) else offsets(new, dev)
    got = paged_append(cache, k, v, table, torch.tensor(lengths, device=dev), q=q, q_offsets=qo, rotary=rotary)
    at = torch.tensor([n - m + i for n, m in zip(lengths, new) for i in range(m)], dtype=torch.int64, device=dev)
    b = [j for j, m in enumerate(new) for _ in range(m)]
    want, bound = turned(q, at, rotary)
    assert bool(((got.cpu().double() - want).abs() <= bound).all())
    pages, slots = table[torch.tensor(b, device=dev), at // page], at % page
    # Rows that no token has are left as they are.
    mask = torch.zeros(cache.values.shape[0], page, dtype=torch.bool, device=dev)
    mask[pages, slots] = True
    kept = (~mask)[:, None, None, :].expand(-1, 2, kv, -1)
    assert torch.equal(cache.values.view(torch.uint8).view(*kept.shape, -1)[kept], before.view(*kept.shape, -1)[kept])
    rows = cache.values[pages, :, :, slots].cpu()
    turned_k, bound = turned(k, at, rotary)
    if store != E4M3:
        assert torch.equal(rows[:, 1], v.cpu())
        assert bool(((rows[:, 0].double() - turned_k).abs() <= bound).all())
        return
    assert torch.equal(cache.scales[kept], scales[kept])
    factors = cache.scales[pages, :, :, slots].cpu().double()
    half = torch.finfo(dtype).eps / 2
    for i, (x, off) in enumerate(((turned_k, (bound - half * turned_k.abs()).clamp_min(0)), (v.cpu().double(), 0.0))):
        top = x.abs().amax(-1)
        off = off + 0.0 * x
        assert bool(((factors[:, i] - top / 448).abs() <= top / 448 * 2.0**-23 + off.amax(-1) / 448).all())
        # Half a step of E4M3: 2^-4 of the value, or 2^-10 of the factor below its normal range; the quotient's rounding.
        err = (rows[:, i].double() * factors[:, i, :, None] - x).abs()
        assert bool((err <= 2.0**-4 * x.abs() * (1 + 2.0**-20) + factors[:, i, :, None] * 2.0**-10 + 2 * off).all())


def test_codes_are_the_row_quantizer_s(dev):
    # Values are not rotated, so that they meet the quantizer as they are: its codes and scales bit for bit.
    cache = PagedCache.zeros(5, 32, 3, 128, E4M3, dev)
    v = make(dev, 130, 3, 128, std=3.0)
    v[7] = 0
    v[9, 1] *= 1e-30
    v[11, 0, 5] = torch.inf
    v[13, 2, 9] = torch.nan
    v[15] = torch.finfo(BF16).max
    table, lengths = torch.arange(5, device=dev)[None], torch.tensor([130], device=dev)
    assert paged_append(cache, v, v, table, lengths, q_offsets=offsets([130], dev)) is None
    codes, scales = kernels.quantize_rows(v.reshape(-1, 128))
    got = cache.values.view(torch.uint8).permute(0, 3, 1, 2, 4).reshape(160, 2, 3, 128)[:130]
    factors = cache.scales.permute(0, 3, 1, 2).reshape(160, 2, 3)[:130]
    for i in range(2):
        assert torch.equal(got[:, i].reshape(-1, 128), codes[:390].view(torch.uint8))
        assert torch.equal(factors[:, i].reshape(-1), scales[:390, 0])


def test_tokens_without_a_place(dev):
    # Padding (length 0), a table that is too short, a page that does not exist, rows outside the offsets.
    rotary = Rotary(rotary_frequencies(64), device=dev)
    for store in (BF16, E4M3):
        cache, _ = pool(dev, [64] * 4, 16, 2, 64, store)
        before = cache.values.view(torch.uint8).clone()
        table = torch.tensor([[0, 1], [2, 3], [4, 99], [-1, 5], [1 << 40, 6]], device=dev)
        lengths = torch.tensor([0, 33, 17, 3, 1], device=dev)
        q, k = make(dev, 5, 4, 64), make(dev, 5, 2, 64)
        got = paged_append(cache, k, k, table, lengths, q=q, rotary=rotary)
        assert not got.any() and torch.equal(cache.values.view(torch.uint8), before)
        # The first two tokens and the last stand outside; the one at 2 is sequence 0's.
        got = paged_append(cache, k, k, table[:1], torch.tensor([9], device=dev), q=q, q_offsets=torch.tensor([2, 3], device=dev),
                           rotary=rotary)
        assert got[2].any() and not got[:2].any() and not got[3:].any()
        changed = (cache.values.view(torch.uint8) != before).flatten(4).any(-1).nonzero()
        assert {(int(a), int(d)) for a, _, _, d in changed} == {(0, 8)}


def test_positions_of_a_model_s_own(dev):
    rotary = Rotary(rotary_frequencies(64), axes=[i % 3 for i in range(32)], device=dev)
    cache, table = pool(dev, [40, 9], 16, 2, 64, BF16)
    q, k = make(dev, 11, 4, 64), make(dev, 11, 2, 64, seed=1)
    at = torch.randint(0, 99, (11, 3), device=dev)
    got = paged_append(cache, k, k, table, torch.tensor([40, 9], device=dev), q=q, q_offsets=offsets([7, 4], dev),
                       rotary=rotary, positions=at)
    want, bound = turned(q, at, rotary)
    assert bool(((got.cpu().double() - want).abs() <= bound).all())
    keys, _ = rows_of(cache, table, [40, 9])
    want, bound = turned(k, at, rotary)
    assert bool(((torch.cat((keys[33:40], keys[45:49])) - want).abs() <= bound).all())


# ---------------------------------------------------------------------------
PROMPTS = [([200], [200]), ([129], [1000]), ([0, 150, 1, 300], [0, 400, 77, 300]), ([700], [900]), ([40, 500, 33], [40, 2000, 500]),
           ([3] * 70 + [300], [9] * 70 + [1100])]
ATTENDS = [([1], [1]), ([1], [77]), ([1, 1, 1], [31, 32, 33]), ([1] * 5, [0, 1, 127, 129, 2000]), ([1], [5000]), ([2, 3], [300, 3]),
           ([5, 1], [5, 900]), ([0, 4, 0, 1], [0, 4, 7, 129]), ([40], [17]), ([63], [130]), ([1] * 70, list(range(70)))]


@pytest.mark.parametrize("heads,kv,dim,dtype,store,page", [
    (8, 2, 128, BF16, BF16, 16), (3, 3, 64, F16, F16, 64), (7, 1, 96, BF16, BF16, 32), (10, 2, 80, F16, F16, 16),
    (8, 2, 128, BF16, E4M3, 16), (32, 8, 128, F16, E4M3, 64), (4, 4, 64, BF16, E4M3, 16), (7, 1, 96, F16, E4M3, 128),
    (10, 2, 80, BF16, E4M3, 32)])
@pytest.mark.parametrize("new,lengths", ATTENDS + PROMPTS, ids=lambda v: "-".join(map(str, v[:6])))
def test_attention(dev, new, lengths, heads, kv, dim, dtype, store, page):
    cache, table = pool(dev, lengths, page, kv, dim, store, seed=len(lengths))
    q = make(dev, sum(new), heads, dim, dtype=dtype, std=2.0)
    qo = None if new == [1] * len(new) else offsets(new, dev)
    got = paged_attention(q, cache, table, torch.tensor(lengths, device=dev), q_offsets=qo)
    attended(cache, q, table, lengths, qo, got)


@pytest.mark.parametrize("dim", [8, 16, 32, 48, 64, 72, 104, 112, 120, 128])
def test_head_dimensions(dev, dim):
    for dtype, store in ((BF16, BF16), (F16, F16)) + (((BF16, E4M3), (F16, E4M3)) if dim % 16 == 0 else ()):
        cache, table = pool(dev, [45, 900], 16, 2, dim, store)
        n = torch.tensor([45, 900], device=dev)
        for new in ([1, 1], [40, 130]):
            q, qo = make(dev, sum(new), 4, dim, dtype=dtype, std=2.0), offsets(new, dev)
            attended(cache, q, table, [45, 900], qo, paged_attention(q, cache, table, n, q_offsets=qo))


@pytest.mark.parametrize("dtype,store", [(BF16, BF16), (F16, F16), (BF16, E4M3), (F16, E4M3)])
@pytest.mark.parametrize("dim,page,new", [(128, 16, 1), (64, 32, 1), (96, 64, 2), (128, 256, 1)])
def test_many_short_sequences(dev, dim, page, new, dtype, store):
    # More tiles than twice what the GPU holds, of up to 256 keys: workgroups of one wave.
    batch, heads = (230, 9) if dim <= 64 else (130, 9)
    rng = random.Random(dim)
    lengths = [rng.choice((0, 1, page - 1, page, rng.randint(1, page))) for _ in range(batch)]
    cache, table = pool(dev, lengths, page, heads, dim, store)
    news = [1] * batch if new == 1 else [min(new, n) for n in lengths]
    qo = None if new == 1 else offsets(news, dev)
    q = make(dev, sum(news), heads, dim, dtype=dtype, std=2.0)
    got = paged_attention(q, cache, table, torch.tensor(lengths, device=dev), q_offsets=qo)
    attended(cache, q, table, lengths, qo, got)


@pytest.mark.parametrize("page", [16, 32, 64, 256, 1024, 4096])
@pytest.mark.parametrize("store", [BF16, E4M3])
def test_pages(dev, page, store):
    lengths = [1, page - 1, page, page + 1, 3 * page + 5, 700]
    cache, table = pool(dev, lengths, page, 2, 64, store, seed=page)
    n = torch.tensor(lengths, device=dev)
    for new in ([1] * 6, [1, 15, page, 100, 70, 300]):
        q, qo = make(dev, sum(new), 4, 64, std=2.0), offsets(new, dev)
        attended(cache, q, table, lengths, qo, paged_attention(q, cache, table, n, q_offsets=qo))


@pytest.mark.parametrize("heads,kv", [(1, 1), (16, 1), (17, 1), (40, 1), (16, 16), (24, 8), (5, 5)])
def test_groups(dev, heads, kv):
    for store in (BF16, E4M3):
        cache, table = pool(dev, [3, 400, 1290], 32, kv, 64, store)
        n = torch.tensor([3, 400, 1290], device=dev)
        for new in ([1, 1, 1], [2, 90, 40]):
            q, qo = make(dev, sum(new), heads, 64, std=2.0), offsets(new, dev)
            attended(cache, q, table, [3, 400, 1290], qo, paged_attention(q, cache, table, n, q_offsets=qo))


@pytest.mark.parametrize("store", [BF16, F16, E4M3])
@pytest.mark.parametrize("nq,n", [(1, 33), (1, 640), (1, 5000), (3, 16000), (1, 16383), (130, 1100), (300, 4000)])
def test_every_key_counts_once(dev, nq, n, store):
    # Queries of zeros weigh all keys alike, and v marks key j by d = j % 128, a quarter of the keys for each
    # key head: an output is a count over n, of at most 32 keys, so that one key more or less is 1 / 32 of it.
    # Values and factors are powers of two, so that nothing but the output (and a count's sum) rounds.
    heads, dim, page = 4, 128, 32
    cache, table = pool(dev, [n], page, heads, dim, store)
    j = torch.arange(n, device=dev)
    v = torch.zeros((n, heads, dim), device=dev, dtype=F16 if store == F16 else BF16)
    v[j, j * heads // n, j % dim] = 1.0
    k = torch.randn((n, heads, dim), device=dev).to(v.dtype)
    lengths = torch.tensor([n], device=dev)
    paged_append(cache, k, v, table, lengths, q_offsets=offsets([n], dev))
    if store == E4M3:
        # Rows of one 1 have the scale 1 / 448: make it 1 / 256 with the code of 256.
        ones = cache.values[:, 1].float() == 448
        cache.values[:, 1] = torch.where(ones, 256.0, 0.0).to(E4M3)
        cache.scales[:, 1] = 1 / 256
    q = torch.zeros((nq, heads, dim), device=dev, dtype=v.dtype)
    got = paged_attention(q, cache, table, lengths, q_offsets=offsets([nq], dev)).double()
    half = torch.finfo(v.dtype).eps / 2
    want = torch.cumsum(v.double(), 0)[n - nq:] / torch.arange(n - nq + 1, n + 1, device=dev)[:, None, None]
    assert bool(((got - want).abs() <= (half + 2.0**-23 * 40) * want + torch.finfo(v.dtype).smallest_normal * half * 2).all())


def test_as_packed_attention(dev):
    # The same tiles of the same keys: the contiguous form's bits, where both take tiles of 16 and split alike.
    n = [700, 2000, 33, 5000]
    cache, table = pool(dev, n, 64, 8, 128, BF16)
    q = make(dev, 4, 32, 128, std=2.0)
    got = paged_attention(q, cache, table, torch.tensor(n, device=dev))
    k, v = (x.to(BF16).to(dev) for x in rows_of(cache, table, n))
    want = attention.packed_attention(q, k, v, offsets([1] * 4, dev), offsets(n, dev), causal=True)
    assert bool(((got - want).abs() <= 2.0**-7 * want.abs() + 1e-3).all())


def test_what_lies_past_a_sequence_is_not_read(dev):
    for store in (BF16, E4M3):
        lengths = [5, 70, 1001]
        cache, table = pool(dev, lengths, 32, 2, 64, store, width=40)
        n = torch.tensor(lengths, device=dev)
        calls = [(make(dev, sum(new), 4, 64, std=2.0), offsets(new, dev)) for new in ([1, 1, 1], [5, 70, 200])]
        wants = [paged_attention(q, cache, table, n, q_offsets=qo) for q, qo in calls]
        own = torch.zeros(cache.values.shape[0], 32, dtype=torch.bool, device=dev)
        for row, m in zip(table.tolist(), lengths):
            for i in range(m):
                own[row[i // 32], i % 32] = True
        foreign = ~own[:, None, None, :].expand(-1, 2, 2, -1)
        cache.values.view(torch.uint8).view(*foreign.shape, -1)[foreign] = 0xff  # NaN in each type
        if cache.scales is not None:
            cache.scales[foreign] = torch.nan
        for (q, qo), want in zip(calls, wants):
            assert torch.equal(paged_attention(q, cache, table, n, q_offsets=qo), want)


def test_pages_that_do_not_exist_count_as_zeros(dev):
    for store in (BF16, E4M3):
        cache, table = pool(dev, [100, 1300], 16, 2, 64, store)
        n = torch.tensor([100, 1300], device=dev)
        calls = [(make(dev, sum(new), 4, 64, std=2.0), offsets(new, dev)) for new in ([1, 1], [80, 150])]
        clean = PagedCache(torch.cat((cache.values.view(torch.uint8), torch.zeros_like(cache.values[:1]).view(torch.uint8)))
                           .view(cache.values.dtype), None if cache.scales is None else
                           torch.cat((cache.scales, torch.zeros_like(cache.scales[:1]))))
        for bad in (-1, cache.values.shape[0], 1 << 31, 1 << 32, -(1 << 63), (1 << 63) - 1):
            table[0, 3] = table[1, 0] = table[1, 44] = bad
            zeros = table.clone()
            zeros[zeros == bad] = cache.values.shape[0]
            for q, qo in calls:
                got, want = (paged_attention(q, c, t, n, q_offsets=qo) for c, t in ((cache, table), (clean, zeros)))
                assert torch.equal(got, want), bad


def test_lengths_outside_the_table(dev):
    cache, table = pool(dev, [64, 1024], 16, 2, 64, BF16)
    for new in ([1, 1], [40, 200]):
        q, qo = make(dev, sum(new), 4, 64), offsets(new, dev)
        full = paged_attention(q, cache, table, torch.tensor([0, 1024], device=dev), q_offsets=qo)
        for n in ([-1, 1025], [-(1 << 63), 1 << 40], [0, (1 << 63) - 1]):
            assert torch.equal(paged_attention(q, cache, table, torch.tensor(n, device=dev), q_offsets=qo), full)
        assert not full[:new[0]].any()


def test_offsets_that_decrease_or_lie_outside(dev):
    # Nothing outside the operands is touched and every row of the output is written.
    rng = random.Random(4)
    rotary = Rotary(rotary_frequencies(64), device=dev)
    for i in range(24):
        batch, tokens, page, width = rng.choice((1, 3, 70)), rng.randint(1, 60) if i % 2 else rng.randint(200, 900), 16, 60
        whole = torch.full((40, 2, 2, page, 64), 7.0, device=dev, dtype=BF16)
        cache = PagedCache(whole[10:30])
        table = torch.randint(-3, 24, (batch, width), device=dev)
        pick = lambda hi: rng.choice((-5, 0, hi, 3 * hi, 1 << 40, rng.randint(0, hi)))  # noqa: E731
        lengths = torch.tensor([pick(page * width) for _ in range(batch)], device=dev)
        qo = torch.tensor([pick(tokens) for _ in range(batch + 1)], device=dev)
        q, k = make(dev, tokens, 4, 64, seed=i), make(dev, tokens, 2, 64, seed=i)
        turned_q = paged_append(cache, k, k, table, lengths, q=q, q_offsets=qo, rotary=rotary)
        got = paged_attention(turned_q, cache, table, lengths, q_offsets=qo)
        torch.cuda.synchronize()
        assert bool(torch.isfinite(got).all()) and bool(torch.isfinite(turned_q).all()), i
        assert bool((whole[:10] == 7).all()) and bool((whole[30:] == 7).all()), i


@pytest.mark.parametrize("store", [BF16, E4M3])
def test_scores_and_scales_far_from_one(dev, store):
    # Large scores (weights of the best keys alone), tiny and huge values.
    lengths = [50, 1500]
    n = torch.tensor(lengths, device=dev)
    for std, size in ((30.0, 1.0), (2.0, 1e30), (2.0, 1e-25)):
        cache, table = pool(dev, lengths, 16, 2, 128, store)
        if store == E4M3:
            cache.scales[:, 1] *= size
        else:
            cache.values[:, 1] *= size
        for new in ([1, 1], [20, 150]):
            q, qo = make(dev, sum(new), 4, 128, std=std), offsets(new, dev)
            for scale in (0.01, 0.3):
                attended(cache, q, table, lengths, qo, paged_attention(q, cache, table, n, q_offsets=qo, scale=scale), scale)


def test_cache_past_32_bit_offsets(dev):
    # Elements pass 2^31 (and their bytes 2^32) before the last pages.
    kv, dim, page = 8, 128, 256
    pages = (1 << 31) // (2 * kv * page * dim) + 40
    cache = PagedCache(torch.empty((pages, 2, kv, page, dim), device=dev, dtype=BF16))
    table = torch.arange(pages - 12, pages, device=dev).flip(0)[None].contiguous()
    lengths, n = torch.tensor([3000], device=dev), 3000
    k, v = make(dev, n, kv, dim), make(dev, n, kv, dim, seed=1)
    paged_append(cache, k, v, table, lengths, q_offsets=offsets([n], dev))
    for new in (1, 60):
        q, qo = make(dev, new, 16, dim, std=2.0), offsets([new], dev)
        check(paged_attention(q, cache, table, lengths, q_offsets=qo), q, k, v, qo, offsets([n], dev), causal=True)


def test_layouts_of_q(dev):
    cache, table = pool(dev, [300, 9], 32, 2, 64, BF16)
    n, q = torch.tensor([300, 9], device=dev), make(dev, 2, 8, 64)
    want = paged_attention(q, cache, table, n)
    for other in (torch.cat((q, q), 1)[:, :8], q.transpose(0, 1).contiguous().transpose(0, 1),
                  torch.nn.functional.pad(q, (0, 3))[..., :64], torch.cat((q.reshape(-1)[:3], q.reshape(-1)))[3:].view(q.shape),
                  torch._neg_view(-q)):
        assert torch.equal(paged_attention(other, cache, table, n), want)


@pytest.mark.parametrize("dtype,store", [(BF16, BF16), (F16, F16), (BF16, E4M3)])
def test_prompts_then_single_tokens(dev, dtype, store):
    # Prompts, drafted tokens and single ones into one cache; a last pass over everything agrees with packed
    # attention over the contiguous sequences.
    heads, kv, dim, page = 8, 2, 128, 16
    rotary = Rotary(rotary_frequencies(dim), device=dev)
    total = [70, 33, 1200]
    cache, table = pool(dev, total, page, kv, dim, store)
    tokens = [make(dev, n, heads + 2 * kv, dim, dtype=dtype, seed=i) for i, n in enumerate(total)]
    done, outs = [0, 0, 0], [[], [], []]
    for step in ([60, 20, 500], [0, 0, 650], [1, 1, 1], [4, 0, 7], [1, 1, 1], [4, 11, 41]):
        parts = [t[a:a + m] for t, a, m in zip(tokens, done, step)]
        done = [a + m for a, m in zip(done, step)]
        q, k, v = torch.cat(parts).split((heads, kv, kv), 1)
        n, qo = torch.tensor(done, device=dev), None if step == [1, 1, 1] else offsets(step, dev)
        q = paged_append(cache, k, v, table, n, q=q, q_offsets=qo, rotary=rotary)
        got = paged_attention(q, cache, table, n, q_offsets=qo)
        attended(cache, q, table, done, qo, got)
        for i, part in enumerate(got.split(step)):
            outs[i].append(part)
    assert done == total
    if store == E4M3:
        return
    from vflash_amd.rotary import rotate

    q, k, v = torch.cat(tokens).split((heads, kv, kv), 1)
    at = torch.cat([torch.arange(n) for n in total]).to(dev)
    q, k = rotate(q, k, at, rotary)
    qo = offsets(total, dev)
    check(torch.cat([torch.cat(o) for o in outs]), q, k, v, qo, qo, causal=True)


def test_a_captured_step_replays_other_lengths_and_pages(dev):
    heads, kv, dim, page = 8, 2, 64, 16
    rotary = Rotary(rotary_frequencies(dim), device=dev)
    for store in (BF16, E4M3):
        cache, table = pool(dev, [1000] * 4, page, kv, dim, store)
        qkv, n = make(dev, 4, heads + 2 * kv, dim), torch.tensor([1000, 1, 30, 500], device=dev)

        def step(cache):
            q, k, v = qkv.split((heads, kv, kv), 1)
            return paged_attention(paged_append(cache, k, v, table, n, q=q, rotary=rotary), cache, table, n)

        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            step(cache)
        torch.cuda.current_stream(dev).wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(cache)
        for lengths in ([1000, 1, 30, 500], [3, 999, 0, 64], [1000] * 4):
            n.copy_(torch.tensor(lengths, device=dev))
            table.copy_(table.roll(1, 0))
            qkv.normal_()
            graph.replay()
            torch.cuda.synchronize()
            twin = PagedCache(cache.values.clone(), None if cache.scales is None else cache.scales.clone())
            assert torch.equal(out, step(twin))
            assert torch.equal(twin.values.view(torch.uint8), cache.values.view(torch.uint8))


def test_a_captured_prompt_replays_other_lengths(dev):
    for store in (BF16, E4M3):
        cache, table = pool(dev, [1000] * 3, 16, 2, 64, store)
        q, n, qo = make(dev, 300, 8, 64), torch.tensor([1000, 100, 30], device=dev), offsets([150, 100, 30], dev)
        paged_attention(q, cache, table, n, q_offsets=qo)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = paged_attention(q, cache, table, n, q_offsets=qo)
        for new, lengths in (([150, 100, 30], [1000, 100, 30]), ([300, 0, 0], [300, 9, 1000]), ([1, 298, 1], [700, 900, 1])):
            n.copy_(torch.tensor(lengths, device=dev))
            qo.copy_(offsets(new, dev))
            q.normal_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, paged_attention(q, cache, table, n, q_offsets=qo))


def test_repeated_calls_and_other_streams_agree(dev):
    for store in (BF16, E4M3):
        lengths = [5000, 20, 900]
        cache, table = pool(dev, lengths, 64, 2, 128, store)
        n = torch.tensor(lengths, device=dev)
        for new in ([1, 1, 1], [300, 4, 90]):
            q, qo = make(dev, sum(new), 8, 128, std=2.0), offsets(new, dev)
            want = paged_attention(q, cache, table, n, q_offsets=qo)
            side = torch.cuda.Stream(dev)
            side.wait_stream(torch.cuda.current_stream(dev))
            with torch.cuda.stream(side):
                got = paged_attention(q, cache, table, n, q_offsets=qo)
            torch.cuda.current_stream(dev).wait_stream(side)
            assert torch.equal(got, want)
            for _ in range(5):
                assert torch.equal(paged_attention(q, cache, table, n, q_offsets=qo), want)


def test_native_host_path(dev):
    # The same bits as the Python wrappers'; None for what those have to decide.
    host = _lib.host()
    r = Rotary(rotary_frequencies(64), device=dev)
    turns = (r.phases, r.axis, r.axes, r.interleaved, r.magnitude)
    none = (None, None, 1, False, 1.0)
    for store in (BF16, E4M3):
        cache, table = pool(dev, [90, 60], 16, 2, 64, store)
        twin = PagedCache(cache.values.clone(), None if cache.scales is None else cache.scales.clone())
        n, qo = torch.tensor([90, 60], device=dev), offsets([3, 9], dev)
        q, k, v = make(dev, 12, 8, 64), make(dev, 12, 2, 64, seed=1), make(dev, 12, 2, 64, seed=2)
        a = (cache.values, cache.scales, table, n, qo, None)
        got, want = host.paged_append(q, k, v, *a, *turns), kernels.paged_append(twin, q, k, v, table, n, qo, r, None)
        assert torch.equal(got, want) and torch.equal(cache.values.view(torch.uint8), twin.values.view(torch.uint8))
        assert host.paged_append(None, k, v, *a, *none) is True
        a = (cache.values, cache.scales, table, n, qo)
        assert torch.equal(host.paged_attention(q, *a, None), kernels.paged_attention(q, cache, table, n, qo, 0.125))
        for args in ((q.cpu(), *a, None), (q.half() if store == BF16 else q.float(), *a, None), (q[..., :32], *a, None), (q[:0], *a, None),
                     (q, *a[:2], table.int(), n, qo, None), (q, *a[:2], table, n[:1], qo, None), (q, *a[:4], qo[:2], None),
                     (q, *a[:4], None, None), (q, *a, -1.0), (q, *a, 1), (q[:, :3], *a, None), (torch.nn.Parameter(q), *a, None),
                     (torch._neg_view(q), *a, None), (q, *a[:2], table.cpu(), n, qo, None)):
            assert host.paged_attention(*args) is None
        b = (cache.values, cache.scales, table, n, qo)
        for args in ((q, k, v, *b, None, *none), (None, k, v, *b, torch.arange(12, device=dev), *none),
                     (q, k, v[:, :1], *b, None, *turns), (q, k, v[:11], *b, None, *turns), (q[:11], k, v, *b, None, *turns),
                     (q, k, v, *b, torch.arange(11, device=dev), *turns), (None, k[:, :1], v[:, :1], *b, None, *none),
                     (q, k, v, cache.values[:0], *b[1:], None, *turns)):
            assert host.paged_append(*args) is None


def test_empty_calls(dev):
    cache, table = pool(dev, [9], 16, 2, 64, BF16)
    none = torch.zeros((0, 1), dtype=torch.int64, device=dev)
    zero = torch.zeros(1, dtype=torch.int64, device=dev)
    q = make(dev, 0, 4, 64)
    assert paged_attention(q, cache, none, zero[:0]).shape == (0, 4, 64)
    # Rows of no sequence.
    assert not paged_attention(make(dev, 3, 4, 64), cache, none, zero[:0], q_offsets=zero).any()
    rotary = Rotary(rotary_frequencies(64), device=dev)
    got = paged_append(cache, q[:, :2], q[:, :2], none, zero[:0], q=q, rotary=rotary)
    assert got.shape == (0, 4, 64)
    empty = PagedCache.zeros(0, 16, 2, 64, device=dev)
    q = make(dev, 1, 4, 64)
    assert not paged_append(empty, q[:, :2], q[:, :2], zero[None], zero + 1, q=q, rotary=rotary).any()
    assert not paged_attention(q, empty, zero[None], zero + 1).any()


def test_autograd_notices_that_a_cache_has_changed(dev):
    cache, table = pool(dev, [9, 9], 16, 2, 64, BF16)
    n, k = torch.tensor([9, 9], device=dev), make(dev, 2, 2, 64)
    for append in (lambda: paged_append(cache, k, k, table, n),
                   lambda: kernels.paged_append(cache, None, k, k, table, n, None, None, None)):
        w = torch.ones((), device=dev, dtype=BF16, requires_grad=True)
        y = (cache.values * w).sum()
        append()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with torch.inference_mode():
        paged_append(PagedCache.zeros(3, 16, 2, 64, device=dev), k, k, table, n)


def test_rotary_of_another_kind_is_refused(dev):
    cache, table = pool(dev, [9], 16, 2, 64, BF16)
    k = make(dev, 1, 2, 64)
    with pytest.raises(ValueError, match="take a Rotary"):
        paged_append(cache, k, k, table, torch.tensor([9], device=dev), rotary=1)
