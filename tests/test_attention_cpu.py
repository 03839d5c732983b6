"""Packed attention without a GPU: refusals, the C entry's contract, and its launches."""

import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fw

from tests.launches import LIBRARY, launches
from vflash_amd import _lib
from vflash_amd.attention import packed_attention

BF16 = torch.bfloat16


def operands(tokens=4, keys=6, heads=4, kv=2, dim=64, dtype=BF16):
    q = torch.zeros((tokens, heads, dim), dtype=dtype)
    k = torch.zeros((keys, kv, dim), dtype=dtype)
    return [q, k, k.clone(), torch.tensor([0, 1, tokens]), torch.tensor([0, 3, keys])]


def test_refusals():
    def refused(match, args, **kwargs):
        with pytest.raises(ValueError, match=match):
            packed_attention(*args, **kwargs)

    refused("gfx950", operands())  # everything else in order
    refused("gfx950", operands(), k_lengths=None, causal=True, scale=0.5)
    a = operands()
    refused("rows, heads, dim", [a[0][0], *a[1:]])
    refused("one type", operands(dtype=torch.float32))
    refused("one type", [a[0], a[1].half(), a[2], *a[3:]])
    refused("one shape", [a[0], a[1], a[2][:-1], *a[3:]])
    refused("one shape", [a[0], a[1][..., :32], a[2][..., :32], *a[3:]])
    refused("multiple of the key heads", operands(heads=5))
    refused("multiple of the key heads", operands(heads=0))
    refused("head dimension", operands(dim=12))
    refused("head dimension", operands(dim=136))
    refused("q_offsets", [*a[:3], a[3].int(), a[4]])
    refused("q_offsets", [*a[:3], a[3][:0], a[4]])
    refused("k_offsets", [*a[:4], a[4][:2]])
    refused("k_offsets", a, k_lengths=torch.tensor([1, 1]))
    refused("k_lengths", [*a[:4], a[4][:2]], k_lengths=torch.tensor([1]))
    refused("k_lengths", [*a[:4], a[4][:2]], k_lengths=torch.tensor([1, 9, 1, 9])[::2])
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        refused("scale", a, scale=scale)
    refused("inference-only", [a[0].requires_grad_(), *a[1:]])


def test_scales_past_binary32():
    # What the kernels multiply by is log2(e) times the scale in binary32: neither infinite nor zero.
    for scale in (2.4e38, 3.39e38, 1e-46):
        assert entry(scale=scale) == _lib.VFLASH_EINVAL
        with pytest.raises(ValueError, match="scale"):
            packed_attention(*operands(), scale=scale)
    with pytest.raises(ValueError, match="gfx950"):
        packed_attention(*operands(), scale=2.35e38)


@pytest.mark.parametrize("tokens,heads,key_heads,taken", [
    (1 << 29, 9, 9, False), (477 * 10**6, 9, 9, False), (475 * 10**6, 9, 9, True), (1 << 29, 64, 64, False),
    (1 << 29, 56, 56, True), (1 << 29, 7, 1, True), (1 << 29, 32 * 32, 32, False),
])
def test_single_tokens_are_counted_in_32_bits(tokens, heads, key_heads, taken):
    # A tile per token and key head (per 16 heads of one), on one line or, for multiples of 8, on eight.
    need = _lib.library().vflash_packed_attention_workspace(tokens, 6, tokens, heads, key_heads, 8)
    assert need == (0 if taken else _lib.VFLASH_EINVAL)
    if not taken:
        change = dict(tokens=tokens, batch=tokens, heads=heads, key_heads=key_heads, dim=8, o_ts=heads * 64)
        assert entry(**change) == _lib.VFLASH_EINVAL


def test_forward_mode_is_refused():
    # A tangent that the kernel would drop, on each operand, gradients recorded or not.
    for recorded in (True, False):
        with torch.set_grad_enabled(recorded), fw.dual_level():
            for i in range(3):
                a = operands()
                a[i] = fw.make_dual(a[i], torch.ones_like(a[i]))
                with pytest.raises(ValueError, match="inference-only"):
                    packed_attention(*a)
    a = operands()
    with pytest.raises(ValueError, match="inference-only"):
        torch.func.jvp(lambda q: packed_attention(q, *a[1:]), (a[0],), (a[0],))


def entry(**change):
    p = ctypes.c_void_p(4096)
    args = dict(q=p, q_ts=256, q_hs=64, k=p, k_ts=128, k_hs=64, v=p, v_ts=128, v_hs=64, f16=0, tokens=4, keys=6, heads=4,
                key_heads=2, dim=64, q_offsets=p, k_offsets=p, k_lengths=None, batch=2, causal=1, scale=0.1, out=p,
                o_ts=256, o_hs=64, workspace=None, workspace_bytes=0, stream=None)
    args.update(change)
    return _lib.library().vflash_packed_attention(*args.values())


@pytest.mark.parametrize("change", [
    dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(q_offsets=None), dict(k_offsets=None),
    dict(q=ctypes.c_void_p(4104)), dict(out=ctypes.c_void_p(4104)), dict(k_lengths=ctypes.c_void_p(4100)),
    dict(tokens=0), dict(tokens=1 << 31), dict(keys=-1), dict(keys=1 << 31), dict(batch=-1), dict(heads=3),
    dict(key_heads=0), dict(dim=0), dict(dim=12), dict(dim=136), dict(q_ts=-8), dict(k_hs=4), dict(k_ts=1 << 23),
    dict(o_hs=56), dict(o_ts=248), dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")),
    dict(keys=100000),  # splits its keys: needs a workspace
    dict(tokens=1 << 30, heads=64, key_heads=64),  # more workgroups than a grid holds
], ids=str)
def test_contract_violations_launch_nothing(change):
    assert entry(**change) == _lib.VFLASH_EINVAL


P = "@4096"
PLANS = [(1, 77, 1, 32, 8, 128), (16, 100000, 16, 32, 8, 128), (1, 131071, 1, 32, 8, 128), (128, 900, 128, 28, 4, 128),
         (500, 500, 24, 28, 4, 128), (8191, 8191, 1, 16, 16, 64), (509, 16509, 1, 32, 8, 128), (40000, 40000, 1, 40, 40, 128),
         (1, 0, 1, 1, 1, 8), (3, 5000, 1, 71, 1, 64), (5000, 60000, 4000, 12, 2, 64), (7, 7, 0, 4, 2, 96), (1, 1, 300, 8, 1, 80)]


@pytest.mark.skipif(not LIBRARY.exists(), reason="the library is not built")
def test_every_tile_has_a_workgroup(tmp_path):
    """A tile is at most 128 (token, head) pairs of one sequence; the grid holds every tile of any
    lengths that the sizes allow, and the split keys' sums fit the workspace."""
    lib = _lib.library()
    calls = []
    for tokens, keys, batch, heads, kv, dim in PLANS:
        # Sized for the stand-in's device of 256 compute units, on which the workspace is at
        # most 2 x 768 + head blocks slots of 128 rows.
        size = (2 * 768 + heads) * 128 * (dim + 2) * 4
        calls.append(("vflash_packed_attention",
                      [P, heads * dim, dim, P, kv * dim, dim, P, kv * dim, dim, 0, tokens, keys, heads, kv, dim, P, P,
                       None, batch, 1, 0.5, P, heads * dim, dim, P, size, None]))
    for plan, (status, run) in zip(PLANS, launches(tmp_path, calls)):
        tokens, keys, batch, heads, kv, dim = plan
        assert status == 0 and 1 <= len(run) <= 2, plan
        kernel, (x, y, z), threads = run[0]
        rows = 16 if kernel.startswith("attention_step") else 128
        group = heads // kv
        per = min(group, rows)
        blocks = kv * -(-group // per)
        worst = min(tokens, tokens // (rows // per) + batch + 2) * blocks
        if rows == 128:
            assert x >= worst and y == z == 1 and threads == 256, plan
        else:  # each workgroup takes its part of all tiles
            assert x % 8 == 0 and x <= 512 and y == z == 1 and threads == 256, plan
        if len(run) == 2:
            name, (jx, jy, _), threads = run[1]
            assert threads == (256 if rows == 128 else 1024)
            assert name.startswith("attention_join") and jx >= worst if rows == 128 else jx == x, plan
    assert lib.vflash_packed_attention_workspace(0, 1, 1, 4, 2, 64) == _lib.VFLASH_EINVAL
