"""The weight-only NVFP4 linear (unquantized activations) against its definition in 64 bits."""

import pytest
import torch
import torch.autograd.forward_ad as fw

from vflash_amd import _lib, kernels
from vflash_amd.nvfp4_linear import NVFP4Execution, NVFP4Weight
from vflash_amd.prepare import quantize_nvfp4_weight

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def restored(packed, scales):
    """The weight's factors e2m1 * e4m3 in 64 bits, from the storage format."""
    n, half = packed.shape
    code = torch.stack((packed & 15, packed >> 4), -1).reshape(n, 2 * half).long()
    value = torch.tensor(E2M1 + [-v for v in E2M1], dtype=torch.float64, device=packed.device)[code]
    tiled = scales.reshape(n // 128, half // 32, 32, 4, 4)  # tile row, tile column, n % 32, n % 128 / 32, block % 4
    block = tiled.permute(0, 3, 2, 1, 4).reshape(n, half // 8).view(torch.float8_e4m3fn).double()
    return value * block.repeat_interleave(16, 1)


def check(got, x, weight, bias):
    """Rounded once to bf16 (half a step, 2^-8), the sum of K products and the two operations
    after it in binary32."""
    x, w, alpha = x.double(), restored(weight.packed, weight.scales), weight.alpha.double()
    want, reach = x @ w.T * alpha, x.abs() @ w.abs().T * alpha
    if bias is not None:
        want, reach = want + bias.double(), reach + bias.double().abs()
    assert got.dtype == BF16 and got.shape == want.shape
    off = 2.0**-24 * (x.shape[1] + 8) * reach
    bound = (want.abs() + off) * 2.0**-8 + off + 2.0**-133
    assert bool(torch.isfinite(got).all())
    worst = ((got.double() - want).abs() - bound).max().item()
    assert worst <= 0, f"{worst} past the bound"


def make(dev, m, n, k, dtype, bias=True, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed + m + n + k)
    x = torch.randn((m, k), generator=g, device=dev).to(dtype)
    w = torch.randn((n, k), generator=g, device=dev) * 0.02
    b = (torch.randn(n, generator=g, device=dev) * 0.1).to(BF16) if bias else None
    return x, NVFP4Weight(*quantize_nvfp4_weight(w)), b


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("m", [1, 2, 3, 15, 16, 17, 31, 33, 64, 65, 127, 130, 256, 257, 300, 513, 1100])
@pytest.mark.parametrize("n,k", [(128, 64), (384, 192), (1152, 1088)])
def test_shapes(dev, m, n, k, dtype):
    for bias in (True, False):
        x, weight, b = make(dev, m, n, k, dtype, bias)
        ex = NVFP4Execution("unquantized")
        check(ex.linear(x, weight, b), x, weight, b)
        assert ex.calls == 1 and ex.rows == m


@pytest.mark.parametrize("m,n,k", [(1, 128, 14336), (1, 16384, 320), (9, 28672, 64), (40, 16384, 128), (700, 2048, 2112),
                                   (33, 256, 9216), (2100, 640, 256)])
def test_long_and_wide(dev, m, n, k):
    for dtype in (BF16, F16):
        x, weight, b = make(dev, m, n, k, dtype)
        check(NVFP4Execution("unquantized").linear(x, weight, b), x, weight, b)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("m", [64, 320])
def test_every_code_times_every_scale(dev, m, dtype):
    # One-hot rows read the weight out: exact in both types, NaN scales as NaN.
    n, k = 512, 64
    g = torch.Generator(device=dev).manual_seed(1)
    packed = torch.randint(0, 256, (n, k // 2), generator=g, device=dev, dtype=torch.uint8)
    scales = torch.arange(n * k // 16, device=dev).to(torch.uint8).reshape(n, k // 16)
    one = torch.ones((), device=dev)
    weight = NVFP4Weight(packed, scales, one, one)
    x = torch.eye(k, device=dev).repeat(m // k, 1).to(dtype)
    got = NVFP4Execution("unquantized").linear(x, weight)
    w = restored(packed, scales)
    # A NaN scale reaches every output of its row (its products with the zeros are NaN too).
    want = torch.where(w.isnan().any(1, keepdim=True), torch.nan, w).T.repeat(m // k, 1)
    assert torch.equal(torch.nan_to_num(got.double(), nan=1e30), torch.nan_to_num(want, nan=1e30))


@pytest.mark.parametrize("m", [1, 5, 40, 300])
def test_rows_do_not_mix(dev, m):
    x, weight, b = make(dev, m, 256, 320, BF16)
    ex = NVFP4Execution("unquantized")
    want = ex.linear(x, weight, b)
    bad = x.clone()
    bad[-1, 5] = torch.nan
    got = ex.linear(bad, weight, b)
    assert torch.equal(got[:-1], want[:-1]) and bool(got[-1].isnan().all())


@pytest.mark.parametrize("m", [1, 20, 290])
def test_layouts_types_and_alignment(dev, m):
    x, weight, b = make(dev, m, 256, 192, BF16)
    ex = NVFP4Execution("unquantized")
    want = ex.linear(x, weight, b)
    wide = torch.full((m, 264), torch.nan, device=dev, dtype=BF16)
    wide[:, 8:200] = x
    assert torch.equal(ex.linear(wide[:, 8:200], weight, b), want)  # a slice, read in place
    odd = torch.full((m, 203), torch.nan, device=dev, dtype=BF16)
    odd[:, 3:195] = x
    assert torch.equal(ex.linear(odd[:, 3:195], weight, b), want)
    assert torch.equal(ex.linear(x.T.contiguous().T, weight, b), want)
    assert torch.equal(ex.linear(x.float(), weight, b), want)  # FP32 enters as BF16
    assert torch.equal(ex.linear(x.reshape(1, m, 192), weight, b)[0], want)
    shifted = torch.cat((b[:1], b))[1:]
    assert torch.equal(ex.linear(x, weight, shifted), want)


def test_large_values_stay_binary32(dev):
    # Sums past binary16's range and far below it.
    for dtype, size in ((F16, 6e4), (BF16, 1e30), (BF16, 1e-30), (F16, 6e-8)):
        for m in (1, 40, 300):
            x, weight, _ = make(dev, m, 128, 256, dtype, bias=False)
            x = (torch.sign(x.float()) * size).to(dtype)
            check(NVFP4Execution("unquantized").linear(x, weight), x, weight, None)


def test_repeated_calls_other_streams_and_graphs(dev):
    for m in (1, 50, 300):
        x, weight, b = make(dev, m, 512, 1088, BF16)
        ex = NVFP4Execution("unquantized")
        want = ex.linear(x, weight, b)
        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            assert torch.equal(ex.linear(x, weight, b), want)
        torch.cuda.current_stream(dev).wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ex.linear(x, weight, b)
        for _ in range(3):
            x.normal_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, ex.linear(x, weight, b))


def test_native_host_path(dev):
    # The same bits as the Python wrapper's; None for what that one has to decide.
    host = _lib.host()
    for m in (1, 30, 300):
        x, w, b = make(dev, m, 256, 192, F16)
        for bias in (b, None):
            want = kernels.nvfp4_w16_gemm(x, w.packed, w.scales, w.alpha, bias)
            assert torch.equal(host.nvfp4_w16_linear(x, w.packed, w.scales, w.alpha, bias), want)
        assert host.nvfp4_w16_linear(x.reshape(1, m, 192), w.packed, w.scales, w.alpha, b).shape == (1, m, 256)
    for args in ((x.float(), w.packed, w.scales, w.alpha, b), (x[:, :64], w.packed, w.scales, w.alpha, b),
                 (x.cpu(), w.packed, w.scales, w.alpha, b), (x, w.packed, w.scales, w.alpha, b[:8]),
                 (x, w.packed, w.scales, w.alpha.cpu(), b), (x.clone().requires_grad_(), w.packed, w.scales, w.alpha, b),
                 (x[:0], w.packed, w.scales, w.alpha, b), (x, w.packed[:64], w.scales[:64], w.alpha, None)):
        assert host.nvfp4_w16_linear(*args) is None


def test_refusals(dev):
    x, weight, b = make(dev, 4, 128, 64, BF16)
    ex = NVFP4Execution("unquantized")
    for args in ((x[:, :32], weight, b), (x.double(), weight, b), (x, weight, b.float()), (x, weight, b[:64]),
                 (x[:0], weight, b), (x.cpu(), weight, b), (x.clone().requires_grad_(), weight, b)):
        with pytest.raises(ValueError):
            ex.linear(*args)
    assert ex.calls == 0 and ex.rows == 0


def test_forward_mode_is_refused(dev):
    x, weight, b = make(dev, 4, 128, 64, BF16)
    ex = NVFP4Execution("unquantized")
    with torch.no_grad(), fw.dual_level():
        for values, bias in ((fw.make_dual(x, torch.ones_like(x)), b), (x, fw.make_dual(b, torch.ones_like(b)))):
            with pytest.raises(ValueError, match="inference-only"):
                ex.linear(values, weight, bias)
    assert ex.calls == 0


@pytest.mark.parametrize("m", [1, 20, 300])
def test_pending_signs(dev, m):
    x, weight, b = make(dev, m, 256, 192, BF16)
    ex = NVFP4Execution("unquantized")
    assert torch.equal(ex.linear(torch._neg_view(x), weight, b), ex.linear(-x, weight, b))
    assert torch.equal(ex.linear(x, weight, torch._neg_view(b)), ex.linear(x, weight, -b))
    twice = NVFP4Weight(weight.packed, weight.scales, torch._neg_view(-weight.alpha), weight.input_scale)
    assert torch.equal(ex.linear(x, twice, b), ex.linear(x, weight, b))


@pytest.mark.parametrize("m", [2, 9, 20, 50, 300])
def test_broadcast_overlapping_and_distant_rows(dev, m):
    x, weight, b = make(dev, m, 256, 192, BF16)
    ex = NVFP4Execution("unquantized")
    flat = torch.randn(16 * m + 192, device=dev).to(BF16)
    distant = torch.zeros(((m - 1) * (1 << 22) + 192,) if m < 20 else (1,), device=dev, dtype=BF16)
    views = [x[:1].expand(m, 192), x[:1].half().expand(m, 192), x[:1].float().expand(m, 192), flat.as_strided((m, 192), (16, 1)),
             x.as_strided((m, 192), (8, 1))]
    if m < 20:
        views.append(distant.as_strided((m, 192), (1 << 22, 1)))
        views[-1].copy_(x)
    for view in views:
        assert torch.equal(ex.linear(view, weight, b), ex.linear(view.contiguous(), weight, b))
    batched = x[:1].expand(m, 192).unflatten(0, (1, m))
    assert torch.equal(ex.linear(batched, weight, b)[0], ex.linear(x[:1].repeat(m, 1), weight, b))
