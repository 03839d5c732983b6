"""The launches of the adapters of many requests that the GPU tests say they reach, for 256 compute units."""

import re

import pytest
import torch

from tests import test_gpu_request_forms as forms
from tests.launches import LIBRARY, launches

pytestmark = pytest.mark.skipif(not LIBRARY.exists(), reason="the library is not built")


def entry(dtype, k, rows, branches, rank):
    n, width = sum(forms.WIDTHS[:branches]), -(-rank // 16) * 16
    # The widths as the 64-bit words of a list of binary32 pairs: their bits, low word first.
    widths = [v for w in forms.WIDTHS[:branches] for v in (torch.tensor(w, dtype=torch.int32).view(torch.float32).item(), 0.0)]
    at = [f"@{4096 + (i << 32)}" for i in range(9)]
    return "vflash_request_adapters", [at[0], n, at[1], k, int(dtype == torch.float16), rows, k, widths, branches, at[2], at[3], at[4],
                                       at[5], 4, width, at[6], at[7], n, at[8], 1 << 40, None]


def test_forms(tmp_path):
    cases, seen = forms.cases(), set()
    for case, (status, run) in zip(cases, launches(tmp_path, [entry(*case) for case in cases])):
        assert status == 0, case
        dtype, k, rows, branches, rank = case
        names = [name for name, _, _ in run]
        assert (names[0] == "request_groups") == (rows > 64), (case, names)
        names = names[rows > 64:]
        f16, width = int(dtype == torch.float16), -(-rank // 16) * 16
        if len(names) == 1:
            assert names == [f"request_few<{f16},{1 if width <= 16 else 2 if width <= 32 else 4}>"], (case, names)
        else:
            all_ranks = branches * width
            assert re.fullmatch(f"request_down<{f16},[14],{4 if all_ranks >= 64 else 2 if all_ranks >= 32 else 1}>", names[0]), (case, names)
            assert names[1:] == [f"request_up<{f16},{1 if width <= 32 else 2 if width <= 64 else 4}>"], (case, names)
        seen.add((rows > 64, *names))
    for f16 in (0, 1):
        for blocks in (1, 2, 4):
            assert {(False, f"request_few<{f16},{blocks}>"), (True, f"request_few<{f16},{blocks}>")} <= seen
        for down, up in ((1, 1), (2, 1), (4, 1), (4, 2), (4, 4)):
            for grouped, rows in ((False, 1), (True, 1), (True, 4)):
                assert (grouped, f"request_down<{f16},{rows},{down}>", f"request_up<{f16},{up}>") in seen, (f16, grouped, rows, down, up)
