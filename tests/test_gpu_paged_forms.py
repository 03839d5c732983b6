"""Every form that paged attention takes (tiles of 16 in workgroups of one, two and four waves, whole and split, tiles of
128, whole and split) in every type, store and width of heads, against its definition in 64 bits.  Which form a
shape takes is checked on the CPU (tests/test_paged_forms_cpu.py), for 256 compute units."""

import math
import random

import pytest
import torch

from tests.attention_reference import packed_attention
from tests.test_gpu_paged import attended, make, offsets, pool, rows_of
from vflash_amd import attention
from vflash_amd.paged import PagedCache, paged_attention

pytestmark = pytest.mark.gpu
BF16, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
TYPES = [(BF16, BF16), (F16, F16), (BF16, E4M3), (F16, E4M3)]
FORMS = ["one wave", "one wave, several", "two waves", "two waves, several", "four waves", "four waves, several", "split",
         "split, several", "split, many", "tiles", "tiles, split"]


def shape(form, dim, store):
    """heads, key heads, page, pages of room, new tokens, lengths."""
    rng = random.Random(f"{form} {dim}")
    held = 256 * (2 if dim <= 64 else 1) * (2 if store == E4M3 else 1)
    several = "several" in form
    if form.startswith("one wave"):
        heads, kv, page, width, batch = 18, 9, 64, 4, 2 * held // 9 + 2
    elif form.startswith("two waves"):
        heads, kv, page, width, batch = 32, 8, 16, 44, held // 8 + 3
    elif form.startswith("four waves"):
        heads, kv, page, width, batch = 6, 2, 32, 16, 5
    elif form == "split, many":
        heads, kv, page, width, batch = 2, 2, 16, 100, 21
    elif form.startswith("split"):
        heads, kv, page, width, batch = 8, 2, 128, 40, 6
    elif form == "tiles":
        heads, kv, page, width, batch = 32, 8, 16, 80, 30
    else:
        heads, kv, page, width, batch = 8, 2, 64, 512, 3
    room = page * width
    most = min(room, 3000)
    if form == "tiles":
        new = [rng.choice((0, 1, 15, 16, 17, 18, 33)) for _ in range(batch - 1)]
        new.append(18 * batch - sum(new))
        assert new[-1] > 0
        lengths = [rng.choice((0, 1, m, m + 1, m + rng.randint(0, 200), m + rng.randint(0, 900))) for m in new]
        lengths[-1] = new[-1] + 300
    elif form == "tiles, split":
        new, lengths = [130, 1, 300], [3000, 900, 2111]
    else:
        lengths = [0, 1, most] + [rng.choice((page - 1, page, page + 1, rng.randint(1, most), rng.randint(1, most)))
                                  for _ in range(batch - 3)]
        new = [(1, 2, 3, 0)[i % 4] for i in range(batch)] if several else [1] * batch
    return heads, kv, page, width, new, lengths


def step_dims(store):
    return (64, 48, 16, 128, 80) if store == E4M3 else (64, 40, 8, 128, 72)


def tile_dims(store):
    return (32, 16, 64, 48, 96, 80, 128, 112) if store == E4M3 else (32, 24, 64, 40, 96, 72, 128, 104)


def cases():
    return [(form, dtype, store, dim) for form in FORMS for dtype, store in TYPES
            for dim in (tile_dims(store) if form.startswith("tiles") else step_dims(store))]


def call(dev, form, dtype, store, dim, std=2.0):
    heads, kv, page, width, new, lengths = shape(form, dim, store)
    cache, table = pool(dev, lengths, page, kv, dim, store, seed=dim, width=width)
    q = make(dev, sum(new), heads, dim, dtype=dtype, std=std)
    return q, cache, table, torch.tensor(lengths, device=dev), None if new == [1] * len(new) else offsets(new, dev), new, lengths


def name(v):
    return str(v).replace("torch.", "").replace(" ", "_")


@pytest.mark.parametrize("form,dtype,store,dim", cases(), ids=name)
def test_form(dev, form, dtype, store, dim):
    q, cache, table, n, qo, new, lengths = call(dev, form, dtype, store, dim)
    got = paged_attention(q, cache, table, n, q_offsets=qo)
    attended(cache, q, table, lengths, qo, got)
    for _ in range(2):
        assert torch.equal(paged_attention(q, cache, table, n, q_offsets=qo), got)


EDGES = [(form, dtype, store, dim) for form in ("one wave", "two waves", "two waves, several", "tiles", "tiles, split")
         for dtype, store in TYPES for dim in (64, 128)]


@pytest.mark.parametrize("form,dtype,store,dim", EDGES, ids=name)
def test_what_lies_past_a_sequence_is_not_read(dev, form, dtype, store, dim):
    q, cache, table, n, qo, new, lengths = call(dev, form, dtype, store, dim)
    want = paged_attention(q, cache, table, n, q_offsets=qo)
    page = cache.values.shape[3]
    own = torch.zeros(cache.values.shape[0], page, dtype=torch.bool)
    for row, m in zip(table.tolist(), lengths):
        for i in range(m):
            own[row[i // page], i % page] = True
    foreign = (~own).to(dev)[:, None, None, :].expand(-1, 2, cache.values.shape[2], -1)
    cache.values.view(torch.uint8).view(*foreign.shape, -1)[foreign] = 0xff  # NaN in each type
    if cache.scales is not None:
        cache.scales[foreign] = torch.nan
    assert torch.equal(paged_attention(q, cache, table, n, q_offsets=qo), want)


@pytest.mark.parametrize("form,dtype,store,dim", EDGES, ids=name)
def test_pages_that_do_not_exist_count_as_zeros(dev, form, dtype, store, dim):
    q, cache, table, n, qo, new, lengths = call(dev, form, dtype, store, dim)
    pages, page = cache.values.shape[0], cache.values.shape[3]
    clean = PagedCache(torch.cat((cache.values.view(torch.uint8), torch.zeros_like(cache.values[:1]).view(torch.uint8)))
                       .view(cache.values.dtype), None if cache.scales is None else
                       torch.cat((cache.scales, torch.zeros_like(cache.scales[:1]))))
    gone = torch.rand(table.shape, generator=torch.Generator().manual_seed(3)).to(dev) < 0.2
    longest = lengths.index(max(lengths))
    gone[longest, (lengths[longest] - 1) // page] = gone[longest, 0] = True
    for bad in (-1, pages, 1 << 32, -(1 << 63), (1 << 63) - 1):
        got = paged_attention(q, cache, torch.where(gone, bad, table), n, q_offsets=qo)
        assert torch.equal(got, paged_attention(q, clean, torch.where(gone, pages, table), n, q_offsets=qo)), bad


@pytest.mark.parametrize("form,dtype,store,dim", EDGES, ids=name)
def test_lengths_outside_the_table(dev, form, dtype, store, dim):
    q, cache, table, n, qo, new, lengths = call(dev, form, dtype, store, dim)
    table = torch.randint(0, cache.values.shape[0], table.shape, device=dev)
    room = table.shape[1] * cache.values.shape[3]
    inside = n.clone()
    inside[0], inside[-1] = 0, room
    want = paged_attention(q, cache, table, inside, q_offsets=qo)
    for low, high in ((-1, room + 1), (-(1 << 63), 1 << 40), (-(1 << 32), (1 << 63) - 1)):
        n = inside.clone()
        n[0], n[-1] = low, high
        assert torch.equal(paged_attention(q, cache, table, n, q_offsets=qo), want)


@pytest.mark.parametrize("form,dtype,store,dim", [e for e in EDGES if e[0] in ("two waves", "tiles", "tiles, split")], ids=name)
@pytest.mark.parametrize("std,size", [(30.0, 1.0), (2.0, 2.0**11), (2.0, 2.0**-10)])
def test_scores_and_values_far_from_one(dev, form, dtype, store, dim, std, size):
    # Weights of the best keys alone; large and small values, the largest inside binary16.
    q, cache, table, n, qo, new, lengths = call(dev, form, dtype, store, dim, std)
    if store == E4M3:
        cache.scales[:, 1] *= size
    else:
        cache.values[:, 1] *= size
    k, v = rows_of(cache, table, lengths)
    for scale in (0.01, 0.3):
        got = paged_attention(q, cache, table, n, q_offsets=qo, scale=scale).cpu().double()
        if store != E4M3:
            k, v = k.to(dtype), v.to(dtype)
        want, bound = packed_attention(q, k, v, torch.arange(len(new) + 1) if qo is None else qo, offsets(lengths, "cpu"), causal=True,
                                       scale=scale)
        # Where the best keys hold a zero, what is left may be of weights that binary32 does not hold.  A weight of bf16 or
        # E4M3 pages carries 2^s, s = -(8 + 1 + log2 of the room), and the row's largest is 2^s or more, so that the sum
        # that normalises them is.  A weight below 2^-126 counts as anything from 0 to itself: 2^(-126 - s) of its value; as
        # does one that a factor takes there, of its code of at most 448.
        room = table.shape[1] * cache.values.shape[3]
        small = 2.0 ** (-126 + 9 + math.ceil(math.log2(room)))
        bound = bound + max(lengths) * small * max(448.0, float(v.abs().max()))
        assert bool(torch.isfinite(got).all())
        assert ((got - want).abs() - bound).max().item() <= 0, scale


@pytest.mark.parametrize("form,dtype,store,dim", EDGES, ids=name)
def test_a_captured_call_replays_other_lengths_and_pages(dev, form, dtype, store, dim):
    q, cache, table, n, qo, new, lengths = call(dev, form, dtype, store, dim)
    table = torch.randint(0, cache.values.shape[0], table.shape, device=dev)
    paged_attention(q, cache, table, n, q_offsets=qo)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_attention(q, cache, table, n, q_offsets=qo)
    rng = random.Random(dim)
    for turn in range(4):
        q.normal_()
        table.copy_(table.roll(1, 0).roll(1, 1))
        n.copy_(torch.tensor(rng.sample(lengths, len(lengths)), device=dev))
        if qo is not None:
            qo.copy_(offsets(rng.sample(new, len(new)), dev))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, paged_attention(q, cache, table, n, q_offsets=qo)), turn


@pytest.mark.parametrize("lengths,heads,kv", [([700, 2000, 33, 5000], 32, 8), ([500, 30, 7], 8, 2), ([300] * 70, 16, 8)])
def test_packed_attention_over_the_same_keys(dev, lengths, heads, kv):
    # The two forms see different room, so that they may split, scale weights and sum differently: each is within the
    # definition's bound, and their difference within twice that.
    cache, table = pool(dev, lengths, 64, kv, 128, BF16)
    q, qo, ko = make(dev, len(lengths), heads, 128, std=2.0), torch.arange(len(lengths) + 1), offsets(lengths, "cpu")
    got = paged_attention(q, cache, table, torch.tensor(lengths, device=dev))
    k, v = (x.to(BF16) for x in rows_of(cache, table, lengths))
    contiguous = attention.packed_attention(q, k.to(dev), v.to(dev), qo.to(dev), ko.to(dev), causal=True)
    want, bound = packed_attention(q, k, v, qo, ko, causal=True)
    for out in (got, contiguous):
        assert bool(((out.cpu().double() - want).abs() <= bound).all())
    assert bool(((got.double() - contiguous.double()).abs().cpu() <= 2 * bound).all())
