"""Rotary positions on the GPU against their definition in 64 bits."""

import math

import pytest
import torch

from vflash_amd import _lib, kernels
from vflash_amd.rotary import Rotary, rotary_frequencies, rotate

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def make(dev, tokens, heads, dim, dtype, seed=0, std=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(tokens, heads, dim, generator=g, device=dev) * std).to(dtype)


def turned(x, positions, rotary):
    """The definition, on the CPU, and a bound on the error of a result rounded once from binary32."""
    x, positions = x.detach().cpu(), positions.cpu()
    pairs, phases = rotary.pairs, rotary.phases.cpu()
    at = positions.reshape(len(positions), -1)
    at = at[:, rotary.axis.cpu()] if rotary.axis is not None else at[:, :1].expand(-1, pairs)
    # position * phase modulo one turn, in 64-bit integers as the definition says.
    angle = (at * phases).double() * 2.0**-64 * 2 * math.pi
    cos, sin = (f(angle)[:, None] * rotary.magnitude for f in (torch.cos, torch.sin))
    y = x.double().clone()
    first, second = ((slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if rotary.interleaved
                     else (slice(0, pairs), slice(pairs, 2 * pairs)))
    a, b = y[..., first].clone(), y[..., second].clone()
    y[..., first], y[..., second] = a * cos - b * sin, a * sin + b * cos
    # A sine is 2^-22 off at most (its phase, its series, its roundings), and two products and a sum round.
    half = torch.finfo(x.dtype).eps / 2
    bound = half * y.abs() + torch.finfo(x.dtype).smallest_normal * half * 2
    reach = (a.abs() + b.abs()) * abs(rotary.magnitude) * 2.0**-21
    bound[..., first] += reach
    bound[..., second] += reach
    bound[..., 2 * pairs:] = 0
    return y, bound


def check(got, x, positions, rotary):
    want, bound = turned(x, positions, rotary)
    assert got.shape == x.shape and got.dtype == x.dtype and got.is_contiguous()
    worst = ((got.cpu().double() - want).abs() - bound).max().item() if got.numel() else 0.0
    assert worst <= 0, f"{worst} past the bound"


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,pairs", [(8, 1), (8, 4), (16, 5), (64, 32), (64, 16), (72, 36), (80, 40), (96, 48), (128, 64),
                                       (128, 30), (128, 63), (200, 100), (256, 128), (256, 37)])
def test_pairs(dev, dim, pairs, layout, dtype):
    rotary = Rotary(rotary_frequencies(2 * pairs), layout=layout, magnitude=1.25, device=dev)
    for tokens, heads, kv in ((1, 1, 1), (5, 7, 3), (37, 40, 8)):
        q, k = make(dev, tokens, heads, dim, dtype), make(dev, tokens, kv, dim, dtype, 1)
        positions = torch.randint(0, 1 << 20, (tokens,), device=dev)
        got = rotate(q, k, positions, rotary)
        check(got[0], q, positions, rotary)
        check(got[1], k, positions, rotary)


@pytest.mark.parametrize("position", [0, 1, -1, 131071, 1000003, (1 << 31) + 7, -(1 << 40) - 3, (1 << 63) - 1, -(1 << 63)])
def test_positions_of_any_size(dev, position):
    rotary = Rotary(rotary_frequencies(128, 5e5), device=dev)
    q = make(dev, 3, 4, 128, F16)
    positions = torch.full((3,), position, device=dev)
    got, none = rotate(q, None, positions, rotary)
    assert none is None
    check(got, q, positions, rotary)
    if position == 0:
        assert torch.equal(got, q)


def test_a_negative_position_turns_back(dev):
    rotary = Rotary(rotary_frequencies(128), layout="interleaved", device=dev)
    q = make(dev, 50, 4, 128, F16)
    positions = torch.arange(50, device=dev) * 1009
    back = rotate(rotate(q, None, positions, rotary)[0], None, -positions, rotary)[0]
    # Two roundings of half a step, of values up to sqrt(2) times a pair's larger one.
    size = q.double().unflatten(-1, (64, 2)).norm(dim=-1, keepdim=True).expand(-1, -1, -1, 2).flatten(-2)
    assert bool(((back.double() - q.double()).abs() <= size * 3 * 2.0**-11).all())


def test_axes(dev):
    axes = [i % 3 for i in range(32)]
    rotary = Rotary(rotary_frequencies(64), axes=axes, device=dev)
    q, k = make(dev, 60, 4, 64, BF16), make(dev, 60, 2, 64, BF16, 1)
    positions = torch.randint(-50, 50, (60, 3), device=dev)
    for at in (positions, positions.t().contiguous().t()):
        got = rotate(q, k, at, rotary)
        check(got[0], q, positions, rotary)
        check(got[1], k, positions, rotary)


@pytest.mark.parametrize("layout", ["merged", "heads first", "expanded", "odd strides", "offset", "negative"])
def test_layouts(dev, layout):
    rotary = Rotary(rotary_frequencies(64), device=dev)
    q, k = make(dev, 30, 8, 64, BF16), make(dev, 30, 2, 64, BF16, 1)
    if layout == "merged":
        q, k = torch.cat((q, k), 1).split((8, 2), 1)
    elif layout == "heads first":
        q, k = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k))
    elif layout == "expanded":
        q, k = q[:1].expand(30, 8, 64), k[:, :1].expand(30, 2, 64)
    elif layout == "odd strides":
        q, k = (torch.nn.functional.pad(x, (0, 3))[..., :64] for x in (q, k))
    elif layout == "offset":
        q, k = (torch.cat((x.reshape(-1)[:3], x.reshape(-1)))[3:].view(x.shape) for x in (q, k))
    else:
        q, k = torch._neg_view(q), torch._neg_view(k)
    positions = torch.arange(30, device=dev)
    got = rotate(q, k, positions, rotary)
    check(got[0], q, positions, rotary)
    check(got[1], k, positions, rotary)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_what_is_not_rotated_comes_back_bit_for_bit(dev, layout):
    # NaN payloads and infinities past the pairs stay, and reach nothing else.
    rotary = Rotary(rotary_frequencies(40), layout=layout, device=dev)
    q = make(dev, 20, 3, 64, BF16)
    clean = q.clone()
    q.view(torch.int16)[..., 40:] = torch.randint(-32768, 32767, (20, 3, 24), device=dev).to(torch.int16)
    nan = q[..., 40:].isnan()
    got = rotate(q, None, torch.arange(20, device=dev), rotary)[0]
    rest, given = got.view(torch.int16)[..., 40:], q.view(torch.int16)[..., 40:]
    assert torch.equal(rest[~nan], given[~nan]) and bool(got[..., 40:][nan].isnan().all())
    assert torch.equal(got[..., :40], rotate(clean, None, torch.arange(20, device=dev), rotary)[0][..., :40])


def test_many_tokens(dev):
    # A workgroup for all heads of a token, and several for a few tokens, give the same bits.
    rotary = Rotary(rotary_frequencies(96), layout="interleaved", device=dev)
    q, k = make(dev, 3000, 24, 96, BF16), make(dev, 3000, 8, 96, BF16, 1)
    positions = torch.arange(3000, device=dev) * 7
    got = rotate(q, k, positions, rotary)
    check(got[0], q, positions, rotary)
    check(got[1], k, positions, rotary)
    for a, b in ((0, 1), (100, 164), (2999, 3000)):
        part = rotate(q[a:b], k[a:b], positions[a:b], rotary)
        assert torch.equal(part[0], got[0][a:b]) and torch.equal(part[1], got[1][a:b])


def test_graph_and_streams(dev):
    rotary = Rotary(rotary_frequencies(128), device=dev)
    q, k = make(dev, 9, 8, 128, BF16), make(dev, 9, 2, 128, BF16, 1)
    positions = torch.arange(9, device=dev)
    want = rotate(q, k, positions, rotary)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = rotate(q, k, positions, rotary)
    torch.cuda.current_stream(dev).wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rotate(q, k, positions, rotary)
    for step in (3, 70000, -5):
        positions.add_(step)
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        want = rotate(q, k, positions, rotary)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_native_host_path(dev):
    # The same bits as the Python wrapper's; None for what that one has to decide.
    host = _lib.host()
    r = Rotary(rotary_frequencies(64), magnitude=1.5, device=dev)
    q, k, at = make(dev, 6, 8, 64, BF16), make(dev, 6, 2, 64, BF16), torch.arange(6, device=dev)
    turns = (r.phases, r.axis, r.axes, r.interleaved, r.magnitude)
    for key in (k, None):
        got, want = host.rotate(q, key, at, *turns), kernels.rotate(q, key, at, r)
        assert torch.equal(got[0], want[0]) and (got[1] is None if key is None else torch.equal(got[1], want[1]))
    assert host.rotate(q, k, at[:, None], *turns) is not None
    for args in ((q.cpu(), k, at), (q, k[:5], at), (q, k, at[:5]), (q, k, at.int()), (q, k, at.cpu()), (q.float(), k.float(), at),
                 (q, k.half(), at), (q[..., :32], k[..., :32], at), (q[:0], k[:0], at[:0]), (q, k, at[:, None].expand(6, 2)),
                 (torch.nn.Parameter(q), k, at), (torch._neg_view(q), k, at), (q, k[..., ::1][:, :, :32], at), (q, k, None)):
        assert host.rotate(*args, *turns) is None, args


def test_no_tokens(dev):
    rotary = Rotary(rotary_frequencies(64), device=dev)
    got = rotate(make(dev, 0, 4, 64, BF16), make(dev, 0, 2, 64, BF16), torch.zeros(0, dtype=torch.int64, device=dev), rotary)
    assert got[0].shape == (0, 4, 64) and got[1].shape == (0, 2, 64)
