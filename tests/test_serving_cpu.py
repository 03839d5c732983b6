"""Rotary positions, the paged cache and the request adapters without a GPU: refusals, the C entries' contracts,
the frequencies and phases, and the launches."""

import ctypes
import math

import pytest
import torch
import torch.autograd.forward_ad as fw

from tests.launches import LIBRARY, launches
from vflash_amd import _lib
from vflash_amd.adapters import RequestAdapters, add_request_adapters, stack_request_adapters
from vflash_amd.fused import LowRankResidual
from vflash_amd.paged import PagedCache, paged_append, paged_attention
from vflash_amd.rotary import Rotary, rotary_frequencies, rotate

BF16, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def refuses(call):
    def refused(match, *args, **kwargs):
        with pytest.raises(ValueError, match=match):
            call(*args, **kwargs)

    return refused


def heads(tokens=4, n=4, dim=64, dtype=BF16):
    return torch.zeros((tokens, n, dim), dtype=dtype)


def turning(pairs=32, **kwargs):
    return Rotary(rotary_frequencies(2 * pairs), device="cpu", **kwargs)


# ---------------------------------------------------------------------------
def test_frequencies():
    f = rotary_frequencies(128, 1e6)
    assert len(f) == 64 and f[0] == 1.0 and math.isclose(f[-1], 1e6 ** (-126 / 128))
    assert rotary_frequencies(128, scaling="linear", factor=4.0) == [x / 4 for x in rotary_frequencies(128)]
    b = rotary_frequencies(128, scaling="base", factor=4.0)
    assert b[0] == 1.0 and math.isclose(b[-1], rotary_frequencies(128)[-1] / 4, rel_tol=1e-12)
    p = rotary_frequencies(128, scaling="parts", factor=8.0, context=4096, low=1.0, high=4.0)
    turns = [4096 * x / (2 * math.pi) for x in rotary_frequencies(128)]
    for x, y, n in zip(p, rotary_frequencies(128), turns):
        assert math.isclose(x, y if n >= 4 else y / 8 if n <= 1 else y * ((n - 1) / 3 + (4 - n) / 3 / 8), rel_tol=1e-12)
    refused = refuses(rotary_frequencies)
    refused("even", 127)
    refused("even", 0)
    refused("positive", 128, 0.0)
    refused("positive", 128, factor=math.inf)
    refused("unknown", 128, scaling="other")
    refused("two pairs", 2, scaling="base", factor=2.0)
    refused("context", 128, scaling="parts", factor=2.0)
    refused("low < high", 128, scaling="parts", factor=2.0, context=100, low=2.0, high=2.0)


def test_phases_are_turns_in_64_bits():
    for f in (1.0, 1e-4, 3.75, -0.5, 2 * math.pi, 1e-30, 12345.678):
        phase = int(Rotary([f], device="cpu").phases[0])
        assert -(2**63) <= phase < 2**63
        for position in (0, 1, -1, 77, 131071, 2**31, -(2**40)):
            turns = (position * phase % 2**64) / 2**64
            # The frequency's own bits, as rationals: 2 pi to 60 digits.
            angle = math.fmod(position * f, 2 * math.pi) if abs(position * f) < 1e6 else None
            if angle is not None:
                far = abs(position * f) * 2.0**-52 + abs(position) * 2.0**-62 + 1e-14
                assert abs(math.sin(turns * 2 * math.pi) - math.sin(angle)) <= far
                assert abs(math.cos(turns * 2 * math.pi) - math.cos(angle)) <= far


def test_rotary_refusals():
    refused = refuses(lambda *a, **k: Rotary(*a, device="cpu", **k))
    refused("layout", [1.0], layout="other")
    refused("finite frequency", [])
    refused("finite frequency", [1.0, math.nan])
    refused("magnitude", [1.0], magnitude=math.inf)
    refused("magnitude", [1.0], magnitude=3.4e38)
    refused("axes", [1.0, 0.5], axes=[0])
    refused("axes", [1.0], axes=[-1])
    refused("axes", [1.0], axes=[64])
    assert turning(axes=[0] * 32).axis is None
    refused, at = refuses(rotate), torch.arange(4)
    refused("gfx950", heads(), heads(n=2), at, turning())  # everything else in order
    refused("gfx950", heads(), None, at[:, None], turning())
    refused("gfx950", heads(dim=256), None, at, turning(128))
    refused("tokens, heads, dim", heads()[0], None, at, turning())
    refused("tokens, heads, dim", heads(n=0), None, at, turning())
    refused("one type", heads(dtype=torch.float32), None, at, turning())
    refused("one type", heads(), heads(dtype=F16), at, turning())
    refused("one head dimension", heads(), heads(dim=72), at, turning())
    refused("multiple of 8", heads(dim=68), None, at, turning())
    refused("multiple of 8", heads(dim=264), None, at, turning())
    refused("same tokens", heads(), heads(tokens=3), at, turning())
    refused("take a Rotary", heads(), None, at, None)
    refused("smaller", heads(), None, at, turning(33))
    refused("int64", heads(), None, at.int(), turning())
    refused("int64", heads(), None, at[:3], turning())
    refused("int64", heads(), None, at, turning(axes=[0, 1] * 16))
    refused("int64", heads(), None, at[:, None].expand(4, 2), turning())
    refused("inference-only", heads().requires_grad_(), None, at, turning())
    with fw.dual_level(), torch.no_grad():
        refused("inference-only", heads(), fw.make_dual(heads(), heads()), at, turning())
    with torch.no_grad():
        refused("gfx950", heads().requires_grad_(), None, at, turning())


# ---------------------------------------------------------------------------
def cache(pages=3, page=16, kv=2, dim=64, dtype=BF16):
    return PagedCache.zeros(pages, page, kv, dim, dtype, device="cpu")


def test_cache_refusals():
    refused, v = refuses(PagedCache), torch.zeros((3, 2, 2, 16, 64), dtype=BF16)
    refused("contiguous", v[:, 0])
    refused("contiguous", torch.zeros((3, 3, 2, 16, 64), dtype=BF16))
    refused("contiguous", v[..., :32])
    for page in (8, 24, 8192):
        refused("power of two", torch.zeros((1, 2, 1, page, 64), dtype=BF16))
    refused("BF16, F16 or E4M3", v.float())
    refused("BF16, F16 or E4M3", v.to(torch.float8_e5m2))
    refused("multiple of 8", torch.zeros((1, 2, 1, 16, 60), dtype=BF16))
    refused("multiple of 8", torch.zeros((1, 2, 1, 16, 136), dtype=BF16))
    refused("multiple of 8", torch.zeros((1, 2, 1, 16, 72)).to(E4M3), torch.ones((1, 2, 1, 16)))
    refused("key heads", torch.zeros((1, 2, 0, 16, 64), dtype=BF16))
    refused("scales", v.to(E4M3))
    refused("scales", v, torch.ones((3, 2, 2, 16)))
    refused("scales", v.to(E4M3), torch.ones((3, 2, 2, 16), dtype=F16))
    refused("scales", v.to(E4M3), torch.ones((3, 2, 2, 15)))
    refused("plain memory", torch.zeros((3, 2, 2, 16, 64), dtype=BF16, requires_grad=True))
    refused("plain memory", torch._neg_view(v))
    refused("plain memory", torch.zeros(3 * 4096 + 1, dtype=BF16)[1:].view(3, 2, 2, 16, 64))


def test_attributes_stay():
    # Their sizes bound what the kernels read: they are not replaced behind the checks.
    c, r = cache(dtype=E4M3), turning(axes=[0, 1] * 16)
    for thing, names in ((c, ("values", "scales")), (r, ("phases", "pairs", "axis", "axes", "interleaved", "magnitude"))):
        for name in names:
            with pytest.raises(AttributeError, match="made of"):
                setattr(thing, name, getattr(thing, name))


TABLE, LENGTHS = torch.zeros((4, 2), dtype=torch.int64), torch.ones(4, dtype=torch.int64)


def test_append_refusals():
    refused = refuses(paged_append)
    k, t, n = heads(n=2), TABLE, LENGTHS
    refused("gfx950", cache(), k, k, t, n)  # everything else in order
    refused("gfx950", cache(dtype=E4M3), k, k, t, n, q=heads(), rotary=turning())
    refused("gfx950", cache(), k, k, t[:2], n[:2], q=heads(), q_offsets=torch.tensor([0, 1, 4]), rotary=turning(),
            positions=torch.arange(4))
    refused("tokens, heads, dim", cache(), k[0], k[0], t, n)
    refused("one type", cache(), k, k.half(), t, n)
    refused("same tokens", cache(), k, k[:3], t, n)
    refused("same tokens", cache(), k, k, t, n, q=heads(3), rotary=turning())
    refused("PagedCache", cache().values, k, k, t, n)
    refused("other heads", cache(kv=1), k, k, t, n)
    refused("other heads", cache(dim=128), k, k, t, n)
    refused("another type", cache(dtype=F16), k, k, t, n)
    refused("page table", cache(), k, k, t.int(), n)
    refused("page table", cache(), k, k, t[0], n)
    refused("page table", cache(), k, k, t[:, :0], n)
    refused("page table", cache(), k, k, t.t().contiguous().t(), n)
    refused("page table", cache(), k, k, torch._neg_view(t), n)
    refused("lengths", cache(), k, k, t, n.int())
    refused("lengths", cache(), k, k, t, n[:3])
    refused("q_offsets", cache(), k, k, t, n, q_offsets=torch.arange(4))
    refused("one token", cache(), heads(3, 2), heads(3, 2), t, n)
    refused("come with rotary", cache(), k, k, t, n, q=heads())
    refused("come with rotary", cache(), k, k, t, n, positions=torch.arange(4))
    refused("take a Rotary", cache(), k, k, t, n, rotary=1)
    refused("smaller", cache(), k, k, t, n, rotary=turning(33))
    refused("several axes", cache(), k, k, t, n, rotary=turning(axes=[0, 1] * 16))
    refused("int64", cache(), k, k, t, n, rotary=turning(), positions=torch.arange(3))
    refused("inference-only", cache(), heads(n=2).requires_grad_(), k, t, n)


def test_attention_refusals():
    refused = refuses(paged_attention)
    q, t, n = heads(), TABLE, LENGTHS
    refused("gfx950", q, cache(), t, n)
    refused("gfx950", q, cache(dtype=E4M3), t[:1], n[:1], q_offsets=torch.tensor([0, 4]), scale=0.5)
    refused("tokens, heads, dim", q[0], cache(), t, n)
    refused("one type", q.float(), cache(), t, n)
    refused("PagedCache", q, None, t, n)
    refused("other heads", q, cache(dim=128), t, n)
    refused("another type", q.half(), cache(), t, n)
    refused("multiple of the key heads", heads(n=5), cache(), t, n)
    refused("page table", q, cache(), t[0], n)
    refused("lengths", q, cache(), t, n[:3])
    refused("one token", heads(5), cache(), t, n)
    for scale in (0.0, -1.0, math.inf, math.nan, 2.4e38, 1e-46):
        refused("scale", q, cache(), t, n, scale=scale)
    refused("inference-only", heads().requires_grad_(), cache(), t, n)


# ---------------------------------------------------------------------------
def residual(rank, k=32, n=48, scaling=0.5, dtype=BF16):
    g = torch.Generator().manual_seed(rank)
    return LowRankResidual(torch.randn((rank, k), generator=g).to(dtype), torch.randn((n, rank), generator=g).to(dtype), scaling)


def test_stack_lays_adapters_side_by_side():
    a, b, c = residual(3), residual(20, n=16), residual(16, n=16)
    pack = stack_request_adapters([(a, None, b), (None, None, None), (None, c, None)], 32, (48, 16, 16), device="cpu")
    assert pack.down.shape == (3, 96, 32) and pack.up.shape == (3, 80, 32) and pack.widths == (48, 16, 16)
    assert pack.ranks.tolist() == [20, 0, 16] and pack.scaling.tolist() == [[0.5, 0, 0.5], [0, 0, 0], [0, 0.5, 0]]
    assert torch.equal(pack.down[0, :3], a.down) and torch.equal(pack.down[0, 64:84], b.down)
    assert torch.equal(pack.up[0, :48, :3], a.up) and torch.equal(pack.up[0, 64:, :20], b.up)
    assert torch.equal(pack.down[2, 32:48], c.down) and torch.equal(pack.up[2, 48:64, :16], c.up)
    assert int(pack.down.count_nonzero()) == 39 * 32 and int(pack.up.count_nonzero()) == 3 * 48 + 36 * 16


def test_stack_refusals():
    refused = refuses(lambda adapters, k=32, widths=(48,): stack_request_adapters(adapters, k, widths, device="cpu"))
    refused("one at least", [])
    refused("for each branch", [(residual(4), None)])
    refused("LowRankResidual", [torch.zeros(3)])
    refused("does not match", [residual(4)], 40)
    refused("does not match", [residual(4)], 32, (56,))
    refused("up to 128", [residual(129)])
    refused("finite", [residual(4, scaling=math.nan)])
    refused("nonempty", [LowRankResidual(torch.zeros((0, 32)), torch.zeros((48, 0)), 1.0)])
    refused("one to three branches", [residual(4, n=12)], 32, (12,))
    refused("one to three branches", [(None,) * 4], 32, (8,) * 4)


def test_adapter_refusals():
    refused = refuses(add_request_adapters)
    pack = stack_request_adapters([residual(4), residual(9)], 32, (48,), device="cpu")
    x, base, index = torch.zeros((5, 32), dtype=BF16), torch.zeros((5, 48), dtype=BF16), torch.zeros(5, dtype=torch.int64)
    refused("gfx950", base, x, pack, index)
    refused("gfx950", base[None], x[None], pack, index, inplace=True)
    refused("RequestAdapters", base, x, pack.down, index)
    refused("does not match", base, x[:, :16], pack, index)
    refused("does not match", base[:, :40], x, pack, index)
    refused("does not match", base[:4], x, pack, index)
    refused("own type", base, x.half(), pack, index)
    refused("own type", base.float(), x, pack, index)
    refused("indices", base, x, pack, index.int())
    refused("indices", base, x, pack, index[:4])
    refused("indices", base, x, pack, torch.zeros(10, dtype=torch.int64)[::2])
    refused("inference-only", base, x.clone().requires_grad_(), pack, index)
    refused("inference-only", base.clone().requires_grad_(), x, pack, index)
    made = refuses(RequestAdapters)
    d, u, s, r = pack.down, pack.up, pack.scaling, pack.ranks
    made("branches", d, u, s, r, ())
    made("one type", d.float(), u.float(), s, r, (48,))
    made("one type", d, u.half(), s, r, (48,))
    made("stacks", d[:0], u[:0], s[:0], r[:0], (48,))
    made("stacks", d[:1], u, s, r, (48,))
    made("padded", d[:, :8], u[..., :8], s, r, (48,))
    made("padded", d, u, s, r, (24, 24))
    made("match the projection", d, u, s, r, (40,))
    made("scaling", d, u, s.double(), r, (48,))
    made("scaling", d, u, s[0], r, (48,))
    made("rank", d, u, s, r.long(), (48,))
    made("contiguous", d.transpose(1, 2).contiguous().transpose(1, 2), u, s, r, (48,))


# ---------------------------------------------------------------------------
P = 4096


def entry(name, change, defaults):
    values = {**defaults, **change}
    assert len(values) == len(defaults)
    return getattr(_lib.library(), name)(*values.values())


ROTATE = dict(q=P, q_ts=256, q_hs=64, k=P, k_ts=128, k_hs=64, f16=0, tokens=4, heads=4, key_heads=2, dim=64, phases=P,
              axis=None, pairs=32, interleaved=0, magnitude=1.0, positions=P, axes=1, q_out=P, k_out=P, stream=None)
APPEND = dict(q=P, q_ts=256, q_hs=64, k=P, k_ts=128, k_hs=64, v=P, v_ts=128, v_hs=64, f16=0, tokens=4, heads=4,
              key_heads=2, dim=64, q_offsets=P, phases=P, axis=None, pairs=32, interleaved=0, magnitude=1.0, positions=None,
              axes=1, values=P, scales=None, pages=3, page=16, table=P, width=2, lengths=P, batch=2, q_out=P, stream=None)
ATTEND = dict(q=P, q_ts=256, q_hs=64, f16=0, tokens=4, heads=4, key_heads=2, dim=64, q_offsets=P, values=P, scales=None,
              pages=3, page=16, table=P, width=2, lengths=P, batch=2, scale=0.125, out=P, o_ts=256, o_hs=64, workspace=None,
              workspace_bytes=0, stream=None)


@pytest.mark.parametrize("name,defaults,changes", [
    ("vflash_rotate", ROTATE, [
        dict(q=None), dict(q=P + 8), dict(q_ts=4), dict(q_hs=-8), dict(k=P + 2), dict(k_out=None), dict(q_out=None), dict(tokens=0),
        dict(tokens=1 << 30), dict(heads=0), dict(heads=65537), dict(key_heads=0), dict(dim=60), dict(dim=264), dict(dim=0),
        dict(phases=None), dict(phases=P + 4), dict(pairs=0), dict(pairs=33), dict(magnitude=math.inf),
        dict(magnitude=math.nan), dict(positions=None), dict(positions=P + 4), dict(axes=0), dict(axes=65), dict(axis=P + 1)]),
    ("vflash_paged_append", APPEND, [
        dict(k=None), dict(v=None), dict(k=P + 8), dict(v_ts=12), dict(q_out=None), dict(phases=None), dict(q_offsets=None),
        dict(q_offsets=P + 4), dict(tokens=0), dict(dim=136), dict(dim=72, scales=P), dict(key_heads=0), dict(key_heads=4097),
        dict(heads=0), dict(values=None), dict(values=P + 8), dict(scales=P + 2), dict(pages=-1), dict(pages=1 << 30),
        dict(page=8), dict(page=24), dict(page=8192), dict(width=0), dict(width=1 << 26), dict(table=None), dict(lengths=None),
        dict(table=P + 4), dict(batch=-1), dict(batch=1 << 30), dict(axes=2), dict(pairs=40)]),
    ("vflash_paged_attention", ATTEND, [
        dict(q=None), dict(q=P + 8), dict(q_ts=4), dict(tokens=0), dict(tokens=1 << 30), dict(heads=5), dict(heads=0),
        dict(key_heads=0), dict(dim=60), dict(dim=136), dict(dim=72, scales=P), dict(q_offsets=None), dict(q_offsets=P + 4),
        dict(values=None), dict(values=P + 8), dict(pages=-1), dict(page=8), dict(page=48), dict(width=0), dict(width=1 << 26),
        dict(table=None), dict(lengths=None), dict(lengths=P + 4), dict(batch=-1), dict(scale=0.0), dict(scale=-1.0),
        dict(scale=math.nan), dict(scale=math.inf), dict(scale=2.4e38), dict(out=None), dict(out=P + 8), dict(o_ts=128),
        dict(o_hs=32), dict(width=64), dict(width=64, workspace=P, workspace_bytes=16)]),
], ids=lambda v: v if isinstance(v, str) else "")
def test_entries_refuse(name, defaults, changes):
    for change in changes:
        assert entry(name, change, defaults) == _lib.VFLASH_EINVAL, change


def test_adapter_entry_refuses():
    widths = (ctypes.c_int64 * 3)(48, 16, 16)
    defaults = dict(base=P, ldb=80, x=P, ldx=32, f16=0, rows=5, k=32, widths=widths, branches=3, down=P, up=P, scaling=P,
                    ranks=P, adapters=2, width=16, index=P, out=P + 4096, ldo=80, workspace=P, workspace_bytes=1 << 20,
                    stream=None)
    for change in (dict(base=None), dict(x=None), dict(down=None), dict(up=None), dict(scaling=None), dict(ranks=None),
                   dict(index=None), dict(out=None), dict(workspace=None), dict(ldb=72), dict(ldb=84), dict(ldx=24),
                   dict(ldx=36), dict(ldo=72), dict(out=P, ldo=88), dict(rows=0), dict(rows=1 << 21), dict(k=0), dict(k=36),
                   dict(widths=None), dict(widths=(ctypes.c_int64 * 3)(48, 12, 16)),
                   dict(widths=(ctypes.c_int64 * 3)(48, 0, 16)), dict(branches=0), dict(branches=4), dict(adapters=0),
                   dict(adapters=8192), dict(width=0), dict(width=24), dict(width=144), dict(workspace_bytes=16),
                   dict(index=P + 4), dict(up=P + 8), dict(ranks=P + 2)):
        assert entry("vflash_request_adapters", change, defaults) == _lib.VFLASH_EINVAL, change


def test_workspaces():
    lib = _lib.library()
    assert lib.vflash_paged_attention_workspace(4, 4, 32, 8, 128, 16, 48, 0) == 0  # room for 768 keys: no split
    assert lib.vflash_paged_attention_workspace(4, 4, 32, 8, 128, 16, 49, 0) > 0
    assert lib.vflash_paged_attention_workspace(4, 4, 32, 8, 128, 17, 49, 0) == _lib.VFLASH_EINVAL
    widths = (ctypes.c_int64 * 1)(64)
    small = lib.vflash_request_adapters_workspace(64, 64, widths, 1, 5, 16)
    assert small == 64 * 16 * 4 + 10 * (4 + 16) * 4  # one part of t, and at most ten items
    assert lib.vflash_request_adapters_workspace(65, 64, widths, 1, 5, 16) > 65 * 16 * 4
    assert lib.vflash_request_adapters_workspace(65, 60, widths, 1, 5, 16) == _lib.VFLASH_EINVAL


def test_launches(tmp_path):
    if not LIBRARY.exists():
        pytest.skip("no library")

    def arguments(defaults, **change):
        return [f"@{v}" if v == P and isinstance(v, int) else v for v in {**defaults, **change}.values()]

    # A workgroup a token; more tokens than a grid's first dimension takes continue in the second.  Few tokens: eight heads
    # of 64 each.
    calls = [("vflash_rotate", arguments(ROTATE)), ("vflash_rotate", arguments(ROTATE, heads=40, key_heads=40)),
             ("vflash_rotate", arguments(ROTATE, tokens=(1 << 22) + 1, f16=1)),
             ("vflash_paged_append", arguments(APPEND)), ("vflash_paged_append", arguments(APPEND, tokens=2, q_offsets=None)),
             ("vflash_paged_attention", arguments(ATTEND)), ("vflash_paged_attention", arguments(ATTEND, scales=P, f16=1)),
             ("vflash_paged_attention", arguments(ATTEND, width=64, workspace=P, workspace_bytes=1 << 30)),
             ("vflash_paged_attention", arguments(ATTEND, tokens=300, batch=300, q_offsets=None, width=128, workspace=P,
                                                  workspace_bytes=1 << 30)),
             ("vflash_paged_attention", arguments(ATTEND, tokens=300, batch=300, q_offsets=None))]
    got = launches(tmp_path, calls)
    assert all(status == 0 for status, _ in got)
    kernels = [[(name, grid) for name, grid, _ in done] for _, done in got]
    assert kernels[0] == [("rotate_heads<0>", (4, 1, 1))] and kernels[1] == [("rotate_heads<0>", (4, 1, 10))]
    assert kernels[2] == [("rotate_heads<1>", (1 << 22, 2, 1))]
    assert kernels[3] == [("rotate_heads<0>", (4, 1, 1))] and kernels[4] == [("rotate_heads<0>", (2, 1, 1))]
    assert [k for k, _ in kernels[5]] == ["attention_step<0,64,1,4>"] and [k for k, _ in kernels[6]] == ["attention_step<1,64,2,4>"]
    assert [k for k, _ in kernels[7]] == ["attention_step<0,64,1,4>", "attention_step_join<0,1,1024>"]
    assert [k for k, _ in kernels[8]] == ["attention_step<0,64,1,4>", "attention_step_join<0,1,256>"]
    assert kernels[9] == [("attention_step<0,64,1,2>", (600, 1, 1))]
