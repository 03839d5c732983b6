"""The adapters of many requests on the GPU against their definition in 64 bits."""

import random

import pytest
import torch

from vflash_amd import _lib, kernels
from vflash_amd.adapters import RequestAdapters, add_request_adapters, stack_request_adapters
from vflash_amd.fused import LowRankResidual

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def make(dev, *shape, dtype=BF16, seed=0, std=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=dev) * std).to(dtype)


def stack(dev, ranks, k, widths, dtype, seed=0):
    """One adapter for each of ``ranks`` (0: none), its branches of different ranks."""
    packs = []
    for i, rank in enumerate(ranks):
        pack = []
        for b, n in enumerate(widths):
            r = max(1, rank - 3 * b)
            pack.append(LowRankResidual(make(dev, r, k, dtype=dtype, seed=seed + 10 * i + b, std=k**-0.5),
                                        make(dev, n, r, dtype=dtype, seed=seed + 500 + 10 * i + b), 0.5 + 0.25 * (i + b) % 3)
                        if rank else None)
        packs.append(tuple(pack))
    return stack_request_adapters(packs, k, widths, dtype=dtype, device=dev)


def defined(base, x, pack, index):
    """The definition on the CPU, and a bound on the error of a result rounded once, whose t has 16 bits or more."""
    base, x = base.cpu().double(), x.cpu().double()
    index = index.cpu().reshape(-1)
    n, k = base.shape[-1], x.shape[-1]
    out, x = base.reshape(-1, n).clone(), x.reshape(-1, k)
    reach = torch.zeros_like(out)
    width = pack.up.shape[2]
    down, up, scaling = pack.down.cpu().double(), pack.up.cpu().double(), pack.scaling.cpu().double()
    for a in range(down.shape[0]):
        rows = (index == a).nonzero()[:, 0]
        first = 0
        for b, w in enumerate(pack.widths):
            d, u = down[a, b * width:(b + 1) * width], up[a, first:first + w]
            out[rows, first:first + w] += scaling[a, b] * (x[rows] @ d.T) @ u.T
            # Sums of k and of the rank round in binary32 (a step each of what they add up in magnitude); t as a high
            # and a low part of 8 bits each loses 2^-16 of its largest value at most (its row's, in binary16).
            t = x[rows].abs() @ d.abs().T
            t = (t * (k * 2.0**-23 + 2.0**-15) + (x[rows] @ d.T).abs().amax(-1, keepdim=True) * 2.0**-15)
            reach[rows, first:first + w] += scaling[a, b].abs() * t @ u.abs().T
            first += w
    half = torch.finfo(pack.down.dtype).eps / 2
    bound = reach + half * out.abs() * (1 + 2.0**-10) + 2.0**-22 * base.reshape(-1, n).abs() + torch.finfo(pack.down.dtype).smallest_normal * half * 2
    return out, bound


def check(got, base, x, pack, index):
    want, bound = defined(base, x, pack, index)
    assert got.shape == base.shape and got.dtype == base.dtype
    got = got.cpu().double().reshape(want.shape)
    assert bool(torch.isfinite(got).all())
    worst = ((got - want).abs() - bound).max().item() if got.numel() else 0.0
    assert worst <= 0, f"{worst} past the bound"


def indices(dev, rows, count, order, seed=0):
    rng = random.Random(seed)
    index = [rng.choice([-1] + [rng.randrange(count)] * 6) for _ in range(rows)]
    return torch.tensor(sorted(index) if order == "runs" else index, device=dev)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("ranks", [[16], [1, 7, 16], [32, 8, 0, 20], [64, 33, 64], [128, 4, 100, 65]], ids=str)
@pytest.mark.parametrize("rows", [1, 2, 16, 17, 63, 64, 65, 200, 513, 700, 1700])
def test_rows_and_ranks(dev, rows, ranks, dtype):
    k, widths = 264, (72,)
    pack = stack(dev, ranks, k, widths, dtype)
    x, base = make(dev, rows, k, dtype=dtype, seed=1), make(dev, rows, 72, dtype=dtype, seed=2)
    for order in ("mixed", "runs"):
        index = indices(dev, rows, len(ranks), order)
        check(add_request_adapters(base, x, pack, index), base, x, pack, index)


@pytest.mark.parametrize("k", [8, 24, 32, 40, 256, 1000, 1024, 5120])
@pytest.mark.parametrize("widths", [(8,), (64,), (136,), (64, 64, 64), (200, 8, 72), (128, 16)], ids=str)
def test_sizes(dev, k, widths):
    for rows in (3, 70):
        pack = stack(dev, [16, 40], k, widths, BF16)
        x, base = make(dev, rows, k, seed=1), make(dev, rows, sum(widths), seed=2)
        index = indices(dev, rows, 2, "mixed")
        check(add_request_adapters(base, x, pack, index), base, x, pack, index)


def test_many_adapters(dev):
    # More adapters than a workgroup has threads, most unused; and every row its own.
    pack = stack(dev, [8] * 1500, 64, (32,), BF16)
    for rows in (50, 300, 1500, 3000):
        x, base = make(dev, rows, 64, seed=1), make(dev, rows, 32, seed=2)
        index = torch.randperm(3000, device=dev)[:rows] % 1500
        check(add_request_adapters(base, x, pack, index), base, x, pack, index)


@pytest.mark.parametrize("rows", [40, 90, 600])
def test_rows_without_an_adapter_keep_their_bits(dev, rows):
    pack = stack(dev, [16, 32], 128, (96,), BF16)
    x, base = make(dev, rows, 128, seed=1), make(dev, rows, 96, seed=2)
    base[3] = torch.nan
    base[5] = torch.inf
    index = torch.randint(0, 2, (rows,), device=dev)
    for i, bad in enumerate((-1, 2, 1 << 31, 1 << 32, -(1 << 63), (1 << 63) - 1, -1, -1)):
        index[i::9] = bad
    none = (index < 0) | (index > 1)
    x[none] = torch.nan  # not read
    got = add_request_adapters(base, x, pack, index)
    assert torch.equal(got.view(torch.int16)[none], base.view(torch.int16)[none])
    want = add_request_adapters(base[~none], x[~none], pack, index[~none])
    assert bool(torch.isfinite(got[~none]).all()) and torch.equal(got[~none], want)
    only = torch.full((rows,), -1, device=dev)
    assert torch.equal(add_request_adapters(base, x, pack, only).view(torch.int16), base.view(torch.int16))


def test_a_row_does_not_depend_on_the_others(dev):
    # A row's bits are its own in any company of one launch form; infinities and NaN of others stay theirs.
    pack = stack(dev, [16, 24, 64], 512, (64, 32), BF16)
    rows = 300
    x, base, index = make(dev, rows, 512, seed=1), make(dev, rows, 96, seed=2), indices(dev, rows, 3, "mixed")
    got = add_request_adapters(base, x, pack, index)
    order = torch.randperm(rows, device=dev)
    assert torch.equal(add_request_adapters(base[order], x[order], pack, index[order]), got[order])
    x2 = x.clone()
    x2[::7] = torch.inf
    x2[3::7] = torch.nan
    fine = torch.ones(rows, dtype=torch.bool, device=dev)
    fine[::7] = fine[3::7] = False
    assert torch.equal(add_request_adapters(base, x2, pack, index)[fine], got[fine])
    for _ in range(3):
        assert torch.equal(add_request_adapters(base, x, pack, index), got)


def test_a_low_rank_of_one_keeps_infinities(dev):
    down, up = torch.zeros((1, 64), device=dev, dtype=F16), torch.ones((16, 1), device=dev, dtype=F16)
    down[0, 0] = 1.0
    pack = stack_request_adapters([LowRankResidual(down, up, 2.0)], 64, (16,), dtype=F16, device=dev)
    x = torch.zeros((3, 64), device=dev, dtype=F16)
    x[0, 0], x[1, 0], x[2, 0] = torch.inf, -torch.inf, 65504.0
    got = add_request_adapters(torch.zeros((3, 16), device=dev, dtype=F16), x, pack, torch.zeros(3, dtype=torch.int64, device=dev))
    # The last is past binary16.
    assert bool((got[0] == torch.inf).all()) and bool((got[1] == -torch.inf).all()) and bool((got[2] == torch.inf).all())


@pytest.mark.parametrize("size", [1024.0, 2.0**-12])
def test_binary16_keeps_t_outside_its_range(dev, size):
    # t near 8e6 and near 5e-7 (of binary16's 65504 and its subnormals), with scalings that bring the result back.
    k = 64
    x, down = ((make(dev, n, k, dtype=F16, seed=n).float() * size).to(F16) for n in (5, 8))
    up = make(dev, 40, 8, dtype=F16, seed=1)
    pack = stack_request_adapters([LowRankResidual(down, up, 1.0 / (8 * size * size))], k, (40,), dtype=F16, device=dev)
    base, index = make(dev, 5, 40, dtype=F16, seed=3), torch.zeros(5, dtype=torch.int64, device=dev)
    check(add_request_adapters(base, x, pack, index), base, x, pack, index)


@pytest.mark.parametrize("rows", [9, 100])
def test_layouts_and_in_place(dev, rows):
    pack = stack(dev, [16, 24], 128, (64, 32), BF16)
    x, base, index = make(dev, rows, 128, seed=1), make(dev, rows, 96, seed=2), indices(dev, rows, 2, "mixed")
    want = add_request_adapters(base, x, pack, index)
    wide = torch.zeros((rows, 200), device=dev, dtype=BF16)
    xs = [x, torch.cat((x, x), 1)[:, 128:], x.t().contiguous().t(), torch.nn.functional.pad(x, (0, 3))[:, :128],
          torch.cat((x.reshape(-1)[:1], x.reshape(-1)))[1:].view(x.shape), torch._neg_view(-x)]
    bases = [base, torch.cat((base, base), 1)[:, 96:], base.t().contiguous().t(), torch.nn.functional.pad(base, (0, 5))[:, :96],
             torch._neg_view(-base)]
    for a in xs:
        assert torch.equal(add_request_adapters(base, a, pack, index), want)
    for b in bases:
        assert torch.equal(add_request_adapters(b, x, pack, index), want)
    wide[:, 8:104] = base
    view = wide[:, 8:104]
    assert add_request_adapters(view, x, pack, index, inplace=True) is view
    assert torch.equal(view, want) and not wide[:, :8].any() and not wide[:, 104:].any()
    own = base.clone()
    assert add_request_adapters(own, x, pack, index, inplace=True) is own and torch.equal(own, want)
    for bad in (base.t().contiguous().t(), torch.nn.functional.pad(base, (0, 5))[:, :96], base[:1].expand(rows, 96), torch._neg_view(-base)):
        with pytest.raises(ValueError, match="in place"):
            add_request_adapters(bad, x, pack, index, inplace=True)
    shaped = add_request_adapters(base.view(1, rows, 96), x.view(1, rows, 128), pack, index.view(1, rows))
    assert shaped.shape == (1, rows, 96) and torch.equal(shaped[0], want)


def test_every_branch_has_its_own(dev):
    # One branch without an adapter, another with a larger rank than the rest.
    k, widths = 96, (64, 24, 40)
    a = LowRankResidual(make(dev, 40, k, std=0.1), make(dev, 24, 40, seed=1), -1.5)
    b = LowRankResidual(make(dev, 3, k, std=0.1, seed=2), make(dev, 64, 3, seed=3), 2.0)
    pack = stack_request_adapters([(None, a, None), (b, None, None), (None, None, None)], k, widths, device=dev)
    x, base = make(dev, 80, k, seed=4), make(dev, 80, 128, seed=5)
    index = torch.arange(80, device=dev) % 4 - 1
    got = add_request_adapters(base, x, pack, index)
    check(got, base, x, pack, index)
    assert torch.equal(got[1::4, :64], base[1::4, :64]) and torch.equal(got[2::4, 64:], base[2::4, 64:])


def test_graph_replays_other_adapters(dev):
    pack = stack(dev, [16, 24, 64], 256, (64,), BF16)
    for rows in (5, 200, 600):
        x, base, index = make(dev, rows, 256, seed=1), make(dev, rows, 64, seed=2), indices(dev, rows, 3, "mixed")
        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            first = add_request_adapters(base, x, pack, index)
        torch.cuda.current_stream(dev).wait_stream(side)
        assert torch.equal(first, add_request_adapters(base, x, pack, index))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = add_request_adapters(base, x, pack, index)
        for seed in range(4):
            index.copy_(indices(dev, rows, 3, "runs" if seed % 2 else "mixed", seed))
            x.normal_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, add_request_adapters(base, x, pack, index))


def test_native_host_path(dev):
    host = _lib.host()
    pack = stack(dev, [16, 24], 128, (64, 32), BF16)
    x, base, index = make(dev, 9, 128, seed=1), make(dev, 9, 96, seed=2), indices(dev, 9, 2, "mixed")
    p = (pack.down, pack.up, pack.scaling, pack.ranks, pack.widths)
    want = kernels.request_adapters(base, x, pack, index, False)
    assert torch.equal(host.request_adapters(base, x, *p, index, False), want)
    own = base.clone()
    assert host.request_adapters(own, x, *p, index, True) is own and torch.equal(own, want)
    for args in ((base.cpu(), x, *p, index, False), (base, x[:8], *p, index, False), (base, x, *p, index.int(), False),
                 (base, x, *p, index[:8], False), (base, x.half(), *p, index, False), (base[:, :88], x, *p, index, False),
                 (base.t().contiguous().t(), x, *p, index, False), (base[:0], x[:0], *p, index[:0], False),
                 (base.clone().requires_grad_(), x, *p, index, False), (base, torch._neg_view(x), *p, index, False),
                 (base, x, *p, index.cpu(), False), (base, x, *p, index, 1), (base[None], x, *p, index, False)):
        assert host.request_adapters(*args) is None


def test_wide_outputs(dev):
    # Outputs whose elements pass 2^31, rows on both sides.
    rows, n = 70000, 32768
    pack = stack(dev, [8], 16, (n,), BF16)
    x = make(dev, rows, 16, seed=1)
    base = torch.zeros((rows, n), device=dev, dtype=BF16)
    index = torch.full((rows,), -1, device=dev)
    index[-3:] = index[5] = 0
    got = add_request_adapters(base, x, pack, index, inplace=True)
    at = [5, 7, rows - 3, rows - 1]
    check(got[at], torch.zeros((4, n), device=dev, dtype=BF16), x[at], pack, index[at])
    assert not got[100:-3].any()


def test_no_rows(dev):
    pack = stack(dev, [8], 32, (16,), BF16)
    none = torch.zeros(0, dtype=torch.int64, device=dev)
    base = torch.zeros((0, 16), device=dev, dtype=BF16)
    assert add_request_adapters(base, torch.zeros((0, 32), device=dev, dtype=BF16), pack, none).shape == (0, 16)
    assert add_request_adapters(base, torch.zeros((0, 32), device=dev, dtype=BF16), pack, none, inplace=True) is base


def test_a_slot_taken_by_another_adapter(dev):
    # Its tensors overwritten in place.
    pack = stack(dev, [16, 24], 64, (48,), BF16)
    other = stack(dev, [9], 64, (48,), BF16, seed=77)
    pack.down[1, :16], pack.up[1, :, :16] = other.down[0], other.up[0]
    pack.down[1, 16:], pack.up[1, :, 16:] = 0, 0
    pack.scaling[1], pack.ranks[1] = other.scaling[0], 9
    x, base, index = make(dev, 20, 64, seed=1), make(dev, 20, 48, seed=2), indices(dev, 20, 2, "mixed")
    check(add_request_adapters(base, x, pack, index), base, x, pack, index)
    assert isinstance(pack, RequestAdapters)


def test_autograd_notices_a_base_changed_in_place(dev):
    pack = stack(dev, [16, 24], 128, (64, 32), BF16)
    x, index = make(dev, 9, 128, seed=1), indices(dev, 9, 2, "mixed")
    for add in (add_request_adapters, lambda b, *a, inplace: kernels.request_adapters(b, *a, inplace)):
        base = make(dev, 9, 96, seed=2)
        w = torch.ones((), device=dev, dtype=BF16, requires_grad=True)
        y = (base * w).sum()
        add(base, x, pack, index, inplace=False)
        before = base._version
        add(base, x, pack, index, inplace=True)
        assert base._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with torch.inference_mode():
        add_request_adapters(make(dev, 9, 96), x, pack, index, inplace=True)


@pytest.mark.parametrize("ranks", [[1, 7, 16], [64, 33, 0]], ids=str)
@pytest.mark.parametrize("rows", [1, 17, 64, 65, 200, 513])
def test_long_inputs(dev, rows, ranks):
    # Two launches and three, where short inputs take one and two.
    pack = stack(dev, ranks, 2056, (200, 72), BF16)
    x, base, index = make(dev, rows, 2056, seed=1), make(dev, rows, 272, seed=2), indices(dev, rows, len(ranks), "mixed")
    check(add_request_adapters(base, x, pack, index), base, x, pack, index)


@pytest.mark.parametrize("rows", [1, 9, 100, 400])
def test_the_input_is_the_base(dev, rows):
    # In place on its own input: nothing of x is read after it was written.
    pack = stack(dev, [16, 24], 1024, (1024,), BF16)
    x, index = make(dev, rows, 1024, seed=1), indices(dev, rows, 2, "mixed")
    want = add_request_adapters(x.clone(), x, pack, index)
    check(want, x, x, pack, index)
    own = x.clone()
    add_request_adapters(own, own, pack, index, inplace=True)
    check(own, x, x, pack, index)
    wide = torch.cat((x, torch.zeros_like(x)), 1)  # the halves overlap in memory, row by row, but not in a value
    add_request_adapters(wide[:, 1024:], wide[:, :1024], pack, index, inplace=True)
    check(wide[:, 1024:], torch.zeros_like(x), x, pack, index)
