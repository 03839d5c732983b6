"""Every launch that the adapters of many requests have (one, two and three kernels, items of 16 and of 64 rows, every
number of rank blocks), in both types, against their definition in 64 bits.  Which a shape takes is checked on the
CPU (tests/test_request_forms_cpu.py), for 256 compute units."""

import pytest
import torch

from tests.test_gpu_request_adapters import check, indices, make, stack
from vflash_amd.adapters import add_request_adapters

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16]
# Branches and the largest rank; the others of its adapters are smaller, one is absent.
RANKS = [(1, 16), (1, 32), (2, 16), (2, 31), (1, 48), (3, 64), (1, 128), (3, 100)]
ROWS = [1, 40, 64, 65, 100, 1700]
INPUTS = [264, 2056]
WIDTHS = (200, 8, 72)


def cases():
    return [(dtype, k, rows, branches, rank) for dtype in TYPES for k in INPUTS for rows in ROWS for branches, rank in RANKS]


@pytest.mark.parametrize("dtype,k,rows,branches,rank", cases(), ids=lambda v: str(v).replace("torch.", ""))
def test_form(dev, dtype, k, rows, branches, rank):
    widths = WIDTHS[:branches]
    pack = stack(dev, [rank, 7, 0, rank - 5], k, widths, dtype)
    x, base = make(dev, rows, k, dtype=dtype, seed=1), make(dev, rows, sum(widths), dtype=dtype, seed=2)
    index = indices(dev, rows, 4, "mixed")
    index[0] = 0
    got = add_request_adapters(base, x, pack, index)
    check(got, base, x, pack, index)
    assert torch.equal(add_request_adapters(base, x, pack, index), got)
    own = base.clone()
    assert add_request_adapters(own, x, pack, index, inplace=True) is own and torch.equal(own, got)
