"""The weight-only NVFP4 linear without a GPU: names, refusals, the C entry's contract, launches."""

import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fw

from tests.launches import LIBRARY, launches
from vflash_amd import _lib
from vflash_amd.nvfp4_linear import NVFP4Execution, NVFP4Weight


def test_names_and_refusals():
    ex = NVFP4Execution("unquantized")
    assert ex.contract == "nvfp4-e2m1-block16-128x4-w4a16-gfx950-v1" and ex.activations == "unquantized"
    assert NVFP4Execution().contract.endswith("w4a4-gfx950-v1")
    assert NVFP4Execution("e4m3").contract.endswith("w4a8-gfx950-v1")
    with pytest.raises(ValueError, match="unquantized"):
        NVFP4Execution("bf16")
    weight = NVFP4Weight(torch.zeros((128, 32), dtype=torch.uint8), torch.zeros((128, 4), dtype=torch.uint8),
                         torch.ones(()), torch.ones(()))
    with pytest.raises(ValueError, match="gfx950"):
        ex.linear(torch.zeros((2, 64), dtype=torch.bfloat16), weight)
    assert ex.calls == 0


def test_forward_mode_is_refused():
    weight = NVFP4Weight(torch.zeros((128, 32), dtype=torch.uint8), torch.zeros((128, 4), dtype=torch.uint8),
                         torch.ones(()), torch.ones(()))
    x, b = torch.zeros((2, 64), dtype=torch.bfloat16), torch.zeros(128, dtype=torch.bfloat16)
    ex = NVFP4Execution("unquantized")
    with torch.no_grad(), fw.dual_level():
        for args in ((fw.make_dual(x, torch.ones_like(x)), weight, b), (x, weight, fw.make_dual(b, torch.ones_like(b)))):
            with pytest.raises(ValueError, match="inference-only"):
                ex.linear(*args)
    assert ex.calls == 0


def entry(**change):
    p = ctypes.c_void_p(4096)
    args = dict(x=p, f16=0, ldx=64, w=p, ws=p, alpha=p, m=4, n=128, k=64, bias=p, out=p, ldo=128, stream=None)
    args.update(change)
    return _lib.library().vflash_nvfp4_w16_linear(*args.values())


@pytest.mark.parametrize("change", [
    dict(x=None), dict(w=None), dict(ws=None), dict(alpha=None), dict(out=None), dict(m=0), dict(n=64), dict(n=192),
    dict(k=32), dict(k=96, ldx=96), dict(ldx=56), dict(ldx=68), dict(ldo=120), dict(ldo=132),
    dict(x=ctypes.c_void_p(4098)), dict(bias=ctypes.c_void_p(4098)), dict(out=ctypes.c_void_p(4104)),
    dict(ldx=1 << 22), dict(k=1 << 24, ldx=1 << 24), dict(n=1 << 25, ldo=1 << 25), dict(m=1 << 31),
    dict(m=(1 << 31) - 1, n=1 << 20, ldo=1 << 20),
], ids=str)
def test_contract_violations_launch_nothing(change):
    assert entry(**change) == _lib.VFLASH_EINVAL


@pytest.mark.skipif(not LIBRARY.exists(), reason="the library is not built")
def test_every_output_has_a_workgroup(tmp_path):
    sizes = [(m, n, k) for m in (1, 16, 17, 64, 65, 256, 257, 1021, 40000) for n in (128, 1152, 16384, 28672)
             for k in (64, 5376)]
    calls = [("vflash_nvfp4_w16_linear", ["@4096", 0, k, "@4096", "@4096", "@4096", m, n, k, None, "@4096", n, None])
             for m, n, k in sizes]
    for (m, n, k), (status, run) in zip(sizes, launches(tmp_path, calls)):
        assert status == 0 and len(run) == 1, (m, n, k)
        kernel, (x, y, z), threads = run[0]
        name, args = kernel.rstrip(">").split("<")
        args = [int(a) for a in args.split(",")]
        if name == "nvfp4_w16_few":
            outputs = 16 * args[1] * 16 * args[2]
            assert threads == 64 * args[5]
        else:
            assert name == "nvfp4_w16_pipe" and threads == 256
            outputs = args[1] * args[2]
        assert x * outputs >= m * n and y == z == 1, (m, n, k)
