"""Packed attention on the GPU against its definition in 64 bits."""

import math
import random

import pytest
import torch
import torch.autograd.forward_ad as fw

from tests.attention_reference import check
from vflash_amd import _lib, kernels
from vflash_amd.attention import packed_attention

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def offsets(lengths, dev):
    return torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int64, device=dev)


def make(dev, nq, nk, heads, kv, dim, dtype, seed=0, std=2.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    q = (torch.randn(sum(nq), heads, dim, generator=g, device=dev) * std).to(dtype)
    k, v = (torch.randn(sum(nk), kv, dim, generator=g, device=dev).to(dtype) for _ in range(2))
    return q, k, v


LENGTHS = [
    ([1], [1]), ([1], [77]), ([1, 1, 1], [31, 32, 33]), ([1] * 5, [0, 1, 127, 129, 2000]), ([1], [5000]),
    ([2, 3], [300, 1]), ([5], [5]), ([64], [64]), ([63, 65], [63, 65]), ([0, 200, 0, 1, 129], [0, 200, 7, 1, 129]),
    ([100], [300]), ([40], [17]), ([130, 33], [0, 500]), ([300], [1100]), ([1, 700], [900, 700]),
]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv,dim,dtype", [(8, 2, 128, BF16), (3, 3, 64, F16), (7, 1, 96, BF16), (10, 2, 80, F16)])
@pytest.mark.parametrize("nq,nk", LENGTHS, ids=lambda v: "-".join(map(str, v)))
def test_lengths(dev, nq, nk, heads, kv, dim, dtype, causal):
    q, k, v = make(dev, nq, nk, heads, kv, dim, dtype)
    qo, ko = offsets(nq, dev), offsets(nk, dev)
    check(packed_attention(q, k, v, qo, ko, causal=causal), q, k, v, qo, ko, causal=causal)


@pytest.mark.parametrize("dim", [8, 16, 24, 32, 40, 56, 72, 88, 104, 112, 120])
@pytest.mark.parametrize("nq,nk", [([1, 1], [45, 200]), ([70], [130])])
def test_head_dimensions(dev, dim, nq, nk):
    for dtype in (BF16, F16):
        q, k, v = make(dev, nq, nk, 4, 2, dim, dtype)
        qo, ko = offsets(nq, dev), offsets(nk, dev)
        check(packed_attention(q, k, v, qo, ko, causal=True), q, k, v, qo, ko, causal=True)


@pytest.mark.parametrize("heads,kv", [(1, 1), (16, 1), (17, 1), (40, 1), (71, 1), (150, 1), (16, 16), (24, 8), (5, 5)])
@pytest.mark.parametrize("nq,nk", [([1, 1, 1], [3, 400, 90]), ([37], [150])])
def test_groups(dev, heads, kv, nq, nk):
    q, k, v = make(dev, nq, nk, heads, kv, 64, BF16)
    qo, ko = offsets(nq, dev), offsets(nk, dev)
    check(packed_attention(q, k, v, qo, ko, causal=True), q, k, v, qo, ko, causal=True)


@pytest.mark.parametrize("nq", [1, 3, 90])
def test_cache_with_room(dev, nq):
    # What lies past a sequence's keys (infinities, NaN) is another's; nothing of it may show.
    lengths, room = [1, 64, 200, 0, 777], 800
    for heads, kv, dim in ((8, 2, 128), (4, 4, 64)):
        q, k, v = make(dev, [nq] * 5, [room] * 5, heads, kv, dim, BF16)
        for i, n in enumerate(lengths):
            k[i * room + n:(i + 1) * room] = torch.inf
            v[i * room + n:(i + 1) * room] = torch.nan
        qo = offsets([nq] * 5, dev)
        ko = torch.arange(5, device=dev) * room
        kl = torch.tensor(lengths, device=dev)
        for causal in (False, True):
            got = packed_attention(q, k, v, qo, ko, k_lengths=kl, causal=causal)
            check(got, q, k, v, qo, ko, k_lengths=kl, causal=causal)
        # Sequences may share rows.
        ko = torch.zeros(5, dtype=torch.int64, device=dev)
        kl = torch.ones(5, dtype=torch.int64, device=dev)
        check(packed_attention(q, k, v, qo, ko, k_lengths=kl), q, k, v, qo, ko, k_lengths=kl)


def test_masked_keys_have_no_weight(dev):
    # Keys that no query sees, or that later queries see, hold infinities and NaN.
    q, k, v = make(dev, [50], [50], 4, 2, 64, BF16)
    qo = offsets([50], dev)
    want = packed_attention(q, k, v, qo, qo, causal=True)
    k[30:] = torch.nan
    got = packed_attention(q, k, v, qo, qo, causal=True)
    assert torch.equal(got[:30], want[:30]) and bool(torch.isnan(got[30:]).all())


def test_rows_outside_every_sequence_are_zeros(dev):
    q, k, v = make(dev, [400], [300], 8, 2, 128, BF16)
    for nq in ([13, 200], [1, 1]):
        qo = torch.tensor([7, 7 + nq[0], 7 + nq[0] + nq[1]], device=dev)
        ko = torch.tensor([0, 100, 300], device=dev)
        got = packed_attention(q, k, v, qo, ko)
        check(got, q, k, v, qo, ko)
        assert not got[:7].any() and not got[7 + sum(nq):].any()


@pytest.mark.parametrize("qo,ko,kl", [
    ([0, -5, 1 << 40], [0, 50, 1 << 40], None), ([0, 60, 30], [-9, 1 << 62, -(1 << 62)], None),
    ([50, 0, 90], [400, 3], [1 << 50, -1]), ([-(1 << 63), 0, (1 << 63) - 1], [299, -4], [5, 1 << 33]),
])
def test_bad_offsets_stay_inside(dev, qo, ko, kl):
    q, k, v = make(dev, [90], [300], 4, 2, 64, BF16)
    t = lambda x: None if x is None else torch.tensor(x, dtype=torch.int64, device=dev)
    got = packed_attention(q, k, v, t(qo), t(ko), k_lengths=t(kl), causal=True)
    torch.cuda.synchronize()
    assert got.shape == q.shape


@pytest.mark.parametrize("tokens,keys,batch,heads,kv", [
    (90, 300, 80, 4, 2), (40, 5000, 5, 8, 4), (150, 100000, 200, 6, 3),  # tiles of 16 rows: whole, split
    (900, 900, 2, 7, 1), (300, 4000, 3, 4, 2), (4000, 5000, 150, 4, 2),  # tiles of 128: whole, split, many sequences
])
def test_bad_offsets_write_every_row_and_no_other(dev, tokens, keys, batch, heads, kv):
    # What lies around the operands is NaN, and must neither show in a row nor change.  The schedule is
    # run on the CPU under the same kinds of offsets (test_attention_schedule_cpu.py).
    dim, room = 64, 64
    g = torch.Generator(device=dev).manual_seed(5)

    def inside(rows, width):
        buffer = torch.full((rows + 2 * room, width, dim), torch.nan, device=dev, dtype=BF16)
        buffer[room:room + rows] = torch.randn((rows, width, dim), generator=g, device=dev).to(BF16)
        return buffer, buffer[room:room + rows]

    (_, q), (_, k), (_, v) = inside(tokens, heads), inside(keys, kv), inside(keys, kv)
    size = _lib.library().vflash_packed_attention_workspace(tokens, keys, batch, heads, kv, dim)
    workspace = torch.full((size // 4 + 256,), torch.nan, device=dev)
    rng = random.Random(tokens)
    for i in range(8):
        def bad(n, hi):
            good = sorted(rng.randint(0, hi) for _ in range(n))
            if i % 4 == 0:
                values = [rng.choice((-(1 << 63), -1, 0, hi, hi + 1, 1 << 32, (1 << 63) - 1, rng.randint(-hi, 2 * hi)))
                          for _ in range(n)]
            elif i % 4 == 1:
                values = good[::-1]
            elif i % 4 == 2:  # falls back once, past the first 64 where there are that many
                values = good[:70] + [x // 2 for x in good[70:]] if n > 70 else good[:1] + [x // 2 for x in good[1:]]
            else:
                values = [x if rng.random() < 0.8 else rng.choice((-5, 3 * hi, rng.randint(0, hi))) for x in good]
            return torch.tensor(values, dtype=torch.int64, device=dev)

        qo, ko = bad(batch + 1, tokens), bad(batch + (i < 4), keys)
        kl = None if i < 4 else bad(batch, keys)
        around, out = inside(tokens, heads)
        out.fill_(torch.nan)
        workspace.fill_(torch.nan)
        _lib.call("vflash_packed_attention", q.data_ptr(), heads * dim, dim, k.data_ptr(), kv * dim, dim, v.data_ptr(),
                  kv * dim, dim, 0, tokens, keys, heads, kv, dim, qo.data_ptr(), ko.data_ptr(),
                  None if kl is None else kl.data_ptr(), batch, i % 2, 0.125, out.data_ptr(), heads * dim, dim,
                  workspace.data_ptr() if size else None, size, _lib.stream_of(dev))
        torch.cuda.synchronize()
        assert bool(torch.isfinite(out).all()), i
        assert bool(around[:room].isnan().all()) and bool(around[room + tokens:].isnan().all()), i
        assert bool(workspace[size // 4:].isnan().all()), i


@pytest.mark.parametrize("layout", ["merged", "heads first", "expanded", "odd strides", "offset"])
@pytest.mark.parametrize("nq", [1, 150])
def test_layouts(dev, layout, nq):
    n, heads, kv, dim = 3, 8, 2, 64
    q, k, v = make(dev, [nq] * n, [nq] * n, heads, kv, dim, F16)
    t = nq * n
    if layout == "merged":
        q, k, v = torch.cat((q, k, v), 1).split((heads, kv, kv), 1)
    elif layout == "heads first":
        q, k, v = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v))
    elif layout == "expanded":
        k, v = k[:1].expand(t, kv, dim), v[:, :1].expand(t, kv, dim)
    elif layout == "odd strides":
        q, k, v = (torch.nn.functional.pad(x, (0, 3))[..., :dim] for x in (q, k, v))
    else:
        q, k, v = (torch.cat((x.reshape(-1)[:3], x.reshape(-1)))[3:].view(x.shape) for x in (q, k, v))
    qo = offsets([nq] * n, dev)
    check(packed_attention(q, k, v, qo, qo, causal=True), q, k, v, qo, qo, causal=True)


def test_scale_and_large_scores(dev):
    q, k, v = make(dev, [1, 70], [600, 70], 4, 2, 128, BF16, std=30.0)
    qo, ko = offsets([1, 70], dev), offsets([600, 70], dev)
    for scale in (1e-6, 0.03, 1.0):
        check(packed_attention(q, k, v, qo, ko, scale=scale), q, k, v, qo, ko, scale=scale)
    # Exponents past binary32's range: the largest score's value alone.
    q = torch.full((1, 1, 64), 1e18, device=dev, dtype=BF16)
    k = torch.ones((200, 1, 64), device=dev, dtype=BF16) * -1.0
    k[123] = -0.5
    v = torch.randn((200, 1, 64), device=dev).to(BF16)
    got = packed_attention(q, k, v, offsets([1], dev), offsets([200], dev))
    assert torch.equal(got[0], v[123])


def test_rows_without_keys_at_large_scales(dev):
    for nq, nk in (([60, 1], [20, 0]), ([1, 2], [300, 1])):
        for dtype in (BF16, F16):
            q, k, v = make(dev, nq, nk, 4, 2, 64, dtype, std=0.2)
            qo, ko = offsets(nq, dev), offsets(nk, dev)
            for scale in (1.0, 40.0):
                check(packed_attention(q, k, v, qo, ko, causal=True, scale=scale), q, k, v, qo, ko, causal=True, scale=scale)


def test_scores_that_rise_and_fall(dev):
    # Later keys far above and far below the first ones, in both types' ranges.
    n = 700
    for dtype, step in ((BF16, 3.0), (F16, 0.1)):
        for sign in (1, -1):
            for nq in (1, 90):
                q, k, v = make(dev, [nq], [n], 2, 1, 64, dtype, std=0.5)
                q[..., 0], k[:, 0, 0] = 1.0, (torch.arange(n, device=dev) * sign * step).to(dtype)
                qo, ko = offsets([nq], dev), offsets([n], dev)
                check(packed_attention(q, k, v, qo, ko, scale=1.0), q, k, v, qo, ko, scale=1.0)


def test_large_values_under_rising_scores(dev):
    # Weights above 1 until the maximum follows: sums of large values stay in binary32.
    n = 700
    for nq in (1, 90):
        q, k, v = make(dev, [nq], [n], 2, 1, 128, BF16, std=0.5)
        q[..., 0], k[:, 0, 0] = 1.0, (torch.arange(n, device=dev) * 0.05).to(BF16)
        v = (v.float() * 1e28).to(BF16)
        qo, ko = offsets([nq], dev), offsets([n], dev)
        check(packed_attention(q, k, v, qo, ko, scale=1.0), q, k, v, qo, ko, scale=1.0)


@pytest.mark.parametrize("nq,n", [(1, 700), (90, 700), (1, 20000), (40, 20000), (300, 3000)])
@pytest.mark.parametrize("step", [0.0, 0.05, -0.05])
@pytest.mark.parametrize("size", [1e-30, 1e36, 3.3895e38], ids=str)
def test_every_finite_value(dev, nq, n, step, size):
    # The sum before its normalisation stays finite up to bf16's largest values, under equal, rising and
    # falling scores, in one part and in several.
    q, k, v = make(dev, [nq], [n], 2, 1, 128, BF16, std=0.5)
    q[..., 0], k[:, 0, 0] = 1.0, ((torch.arange(n, device=dev) % 700) * step).to(BF16)
    if step == 0.0:
        q.zero_()
    v = (v.sign() * size).to(BF16)
    v[:, :, :8] = size
    qo, ko = offsets([nq], dev), offsets([n], dev)
    check(packed_attention(q, k, v, qo, ko, scale=1.0), q, k, v, qo, ko, scale=1.0)


def test_binary16_keeps_small_probabilities(dev):
    # One score 17 above 60000 equal ones: each of these weighs 2^-24.5, together 2.5e-3.
    n = 60000
    q = torch.zeros((1, 1, 64), device=dev, dtype=F16)
    q[..., 0] = 1.0
    k = torch.zeros((n, 1, 64), device=dev, dtype=F16)
    k[4, 0, 0] = 17.0
    v = torch.ones((n, 1, 64), device=dev, dtype=F16)
    v[4] = 0
    qo, ko = offsets([1], dev), offsets([n], dev)
    check(packed_attention(q, k, v, qo, ko, scale=1.0), q, k, v, qo, ko, scale=1.0)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("n", [700, 5000])
@pytest.mark.parametrize("nq", [1, 40])
def test_weights_are_normalised_as_rounded(dev, nq, n, dtype):
    # Every 32nd key weighs 1, the others just below the middle of two 16-bit numbers, so that all of them
    # round down by half a step; a value that the keys share comes back exactly all the same.
    half = torch.finfo(dtype).eps / 2
    weight = 0.5 * (1 + half) * (1 - half / 16)
    q = torch.zeros((nq, 1, 64), device=dev, dtype=dtype)
    q[..., 0] = 1.0
    k = torch.full((n, 1, 64), -1.0, device=dev, dtype=dtype)
    k[::32] = 0.0
    v = torch.full((n, 1, 64), 1.0, device=dev, dtype=dtype)
    got = packed_attention(q, k, v, offsets([nq], dev), offsets([n], dev), scale=-math.log(weight))
    assert torch.equal(got, torch.ones_like(got))


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("nq,n", [(1, 33), (1, 640), (1, 5000), (3, 16000), (1, 16383), (40, 5000), (130, 1100), (300, 4000)])
def test_every_key_counts_once(dev, nq, n, dtype):
    # Queries of zeros weigh all keys alike, and v marks key j by d = j % 128, a quarter of the keys for each
    # key head: an output is a count over n, of at most 32 keys, so that one key more or less is 1 / 32 of
    # it.  Off by its one rounding (half a step) and the sums' binary32.
    heads, dim = 4, 128
    q = torch.zeros((nq, heads, dim), device=dev, dtype=dtype)
    k = torch.randn((n, heads, dim), device=dev).to(dtype)
    j = torch.arange(n, device=dev)
    v = torch.zeros((n, heads, dim), device=dev, dtype=dtype)
    v[j, j * heads // n, j % dim] = 1.0
    got = packed_attention(q, k, v, offsets([nq], dev), offsets([n], dev)).double()
    want = (v.double().sum(0) / n).expand(nq, heads, dim)
    half = torch.finfo(dtype).eps / 2
    assert bool(((got - want).abs() <= (half + 2.0**-23 * 40) * want + torch.finfo(dtype).smallest_normal * half * 2).all())
    # Causal: query i of nq sees n - nq + i + 1 keys.
    got = packed_attention(q, k, v, offsets([nq], dev), offsets([n], dev), causal=True).double()
    seen = torch.cumsum(v.double(), 0)[n - nq:]
    want = seen / torch.arange(n - nq + 1, n + 1, device=dev)[:, None, None]
    assert bool(((got - want).abs() <= (half + 2.0**-23 * 40) * want + torch.finfo(dtype).smallest_normal * half * 2).all())


def test_many_sequences(dev):
    # More sequences than a wave has lanes, long ones among short.
    g = torch.Generator().manual_seed(3)
    for nq in ([1] * 200, torch.randint(0, 40, (150,), generator=g).tolist()):
        nk = [n + (2000 if i % 50 == 7 else i % 9) for i, n in enumerate(nq)]
        q, k, v = make(dev, nq, nk, 4, 2, 64, BF16)
        qo, ko = offsets(nq, dev), offsets(nk, dev)
        check(packed_attention(q, k, v, qo, ko, causal=True), q, k, v, qo, ko, causal=True)


def test_cache_past_32_bit_offsets(dev):
    rows, kv, dim = (1 << 31) // 256 + 5000, 2, 128  # elements pass 2^31 before the last rows
    k = torch.empty((rows, kv, dim), device=dev, dtype=BF16)
    v = torch.empty_like(k)
    for nq in (1, 40):
        q, k[-3000:], v[-3000:] = make(dev, [nq], [3000], 4, kv, dim, BF16)
        qo = offsets([nq], dev)
        got = packed_attention(q, k, v, qo, torch.tensor([rows - 3000], device=dev),
                               k_lengths=torch.tensor([3000], device=dev), causal=True)
        check(got, q, k[-3000:], v[-3000:], qo, torch.tensor([0, 3000]), causal=True)


def test_repeated_calls_and_other_streams_agree(dev):
    for nq, nk in (([1] * 3, [5000, 20, 900]), ([300, 4], [4000, 4])):
        q, k, v = make(dev, nq, nk, 8, 2, 128, BF16)
        qo, ko = offsets(nq, dev), offsets(nk, dev)
        want = packed_attention(q, k, v, qo, ko, causal=True)
        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            got = packed_attention(q, k, v, qo, ko, causal=True)
        torch.cuda.current_stream(dev).wait_stream(side)
        assert torch.equal(got, want)
        for _ in range(5):
            assert torch.equal(packed_attention(q, k, v, qo, ko, causal=True), want)


def test_graph_replays_other_lengths(dev):
    # The lengths are read on the device: a captured call serves others.
    q, k, v = make(dev, [1] * 4, [1000] * 4, 8, 2, 128, BF16)
    qo, ko = offsets([1] * 4, dev), torch.arange(4, device=dev) * 1000
    kl = torch.tensor([1000, 1, 30, 500], device=dev)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        packed_attention(q, k, v, qo, ko, k_lengths=kl)
    torch.cuda.current_stream(dev).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = packed_attention(q, k, v, qo, ko, k_lengths=kl)
    for lengths in ([1000, 1, 30, 500], [3, 999, 0, 64], [1000] * 4):
        kl.copy_(torch.tensor(lengths, device=dev))
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, packed_attention(q, k, v, qo, ko, k_lengths=kl))


def test_native_host_path(dev):
    # The same bits as the Python wrapper's; None for what that one has to decide.
    host = _lib.host()
    q, k, v = make(dev, [1, 60], [90, 60], 8, 2, 64, BF16)
    qo, ko = offsets([1, 60], dev), offsets([90, 60], dev)
    kl = torch.tensor([90, 60], device=dev)
    for causal, scale in ((True, None), (False, 0.3)):
        want = kernels.packed_attention(q, k, v, qo, ko, None, causal, 0.125 if scale is None else scale)
        assert torch.equal(host.packed_attention(q, k, v, qo, ko, None, causal, scale), want)
        assert torch.equal(host.packed_attention(q, k, v, qo, ko[:2], kl, causal, scale), want)
    p = torch.nn.Parameter(q)
    assert host.packed_attention(p, k, v, qo, ko, None, True, None) is None
    with torch.no_grad():
        assert torch.equal(packed_attention(p, k, v, qo, ko), packed_attention(q, k, v, qo, ko))
    for args in ((q.cpu(), k, v, qo, ko, None, True, None), (q, k, v, qo.int(), ko, None, True, None),
                 (q, k, v, qo, ko, kl, True, None), (q, k, v[..., :32], qo, ko, None, True, None),
                 (q, k, v, qo.cpu(), ko, None, True, None), (q, k, v, qo, ko, None, 1, None),
                 (q, k, v, qo, ko, None, True, -1.0), (q, k, v, qo, ko, None, True, 1),
                 (q[:, :3], k, v, qo, ko, None, True, None), (q[:0], k, v, qo, ko, None, True, None),
                 (q.float(), k.float(), v.float(), qo, ko, None, True, None)):
        assert host.packed_attention(*args) is None


def test_pending_signs(dev):
    # torch._neg_view and the imaginary part of a conjugate: the memory holds the opposite sign.
    q, k, v = make(dev, [1, 60], [90, 60], 8, 2, 64, BF16)
    qo, ko = offsets([1, 60], dev), offsets([90, 60], dev)
    for i in range(3):
        a, b = [q, k, v], [q, k, v]
        a[i], b[i] = torch._neg_view(a[i]), -a[i]
        assert torch.equal(packed_attention(*a, qo, ko, causal=True), packed_attention(*b, qo, ko, causal=True))


def test_forward_mode_is_refused(dev):
    q, k, v = make(dev, [4], [9], 4, 2, 64, BF16)
    qo, ko = offsets([4], dev), offsets([9], dev)
    with torch.no_grad(), fw.dual_level():
        for i in range(3):
            a = [q, k, v]
            a[i] = fw.make_dual(a[i], torch.ones_like(a[i]))
            assert _lib.host().packed_attention(*a, qo, ko, None, True, None) is None
            with pytest.raises(ValueError, match="inference-only"):
                packed_attention(*a, qo, ko, causal=True)
        assert _lib.host().packed_attention(q, k, v, qo, ko, None, True, None) is not None


def test_no_rows(dev):
    q, k, v = make(dev, [0], [9], 4, 2, 64, BF16)
    zero = torch.zeros(2, dtype=torch.int64, device=dev)
    assert packed_attention(q, k, v, zero, zero).shape == (0, 4, 64)
    q, k, v = make(dev, [5], [0], 4, 2, 64, BF16)
    assert not packed_attention(q, k, v, offsets([5], dev), zero).any()
    assert not packed_attention(q, k, v, zero[:1], zero[:1]).any()  # no sequence at all
