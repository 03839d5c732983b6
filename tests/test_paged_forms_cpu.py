"""The forms of paged attention that the GPU tests say they reach: what the library launches for their shapes on 256
compute units, so that a changed rule cannot leave one of them without a test of its values."""

import pytest

from tests import test_gpu_paged_forms as forms
from tests.launches import LIBRARY, launches

pytestmark = pytest.mark.skipif(not LIBRARY.exists(), reason="the library is not built")
P = "@4096"


def entry(form, dtype, store, dim):
    heads, kv, page, width, new, lengths = forms.shape(form, dim, store)
    tokens, batch = sum(new), len(new)
    return "vflash_paged_attention", [
        P, heads * dim, dim, int(dtype == forms.F16), tokens, heads, kv, dim, None if new == [1] * batch else P, P,
        P if store == forms.E4M3 else None, 1000, page, P, width, P, batch, 0.125, P, heads * dim, dim, P, 1 << 40, None]


def expected(form, dtype, store, dim):
    f16, stored = int(dtype == forms.F16), 2 if store == forms.E4M3 else 1
    if form.startswith("tiles"):
        tiles = f"attention_tiles<{f16},{-(-dim // 32) * 32},4,{stored}>"
        return [tiles, f"attention_join<{f16},1>"] if "split" in form else [tiles]
    waves = 1 if form.startswith("one") else 2 if form.startswith("two") else 4
    step = f"attention_step<{f16},{64 if dim <= 64 else 128},{stored},{waves}>"
    if not form.startswith("split"):
        return [step]
    return [step, f"attention_step_join<{f16},1,{256 if form == 'split, many' else 1024}>"]


def test_forms(tmp_path):
    cases = forms.cases()
    seen = set()
    for case, (status, run) in zip(cases, launches(tmp_path, [entry(*case) for case in cases])):
        assert status == 0 and [kernel for kernel, _, _ in run] == expected(*case), (case, status, run)
        seen.add((*(kernel for kernel, _, _ in run),))
    # Every instance that the library launches over pages, whole and split.
    for f16 in (0, 1):
        for stored in (1, 2):
            for width in (32, 64, 96, 128):
                tiles = f"attention_tiles<{f16},{width},4,{stored}>"
                assert {(tiles,), (tiles, f"attention_join<{f16},1>")} <= seen
            for width in (64, 128):
                for waves in (1, 2, 4):
                    assert (f"attention_step<{f16},{width},{stored},{waves}>",) in seen
                for threads in (256, 1024):
                    assert (f"attention_step<{f16},{width},{stored},4>", f"attention_step_join<{f16},1,{threads}>") in seen
    assert len(seen) == 4 * (4 * 2 + 2 * (3 + 2))
    # The tests of edges: the same shapes.
    assert set(forms.EDGES) <= set(cases)
