"""What a serving step keeps can be copied, deep-copied and pickled, as the modules that hold it are."""

import copy
import io
import pickle

import pytest
import torch

from vflash_amd.adapters import RequestAdapters, stack_request_adapters
from vflash_amd.fused import LowRankResidual
from vflash_amd.paged import PagedCache
from vflash_amd.rotary import Rotary, _rotary_of, rotary_frequencies


def through_pickle(thing):
    return pickle.loads(pickle.dumps(thing))


def through_save(thing):
    file = io.BytesIO()
    torch.save(thing, file)
    file.seek(0)
    return torch.load(file, weights_only=False)


COPIES = [copy.copy, copy.deepcopy, through_pickle, through_save]


class Holder(torch.nn.Module):
    def __init__(self, thing):
        super().__init__()
        self.thing = thing


@pytest.mark.parametrize("made", COPIES, ids=lambda f: f.__name__)
@pytest.mark.parametrize("kwargs", [{}, dict(layout="interleaved", magnitude=1.25), dict(axes=[0, 1, 2, 0] * 8)], ids=str)
def test_rotary(made, kwargs):
    one = Rotary(rotary_frequencies(64), device="cpu", **kwargs)
    for two in (made(one), made(Holder(one)).thing):
        assert type(two) is Rotary and (made is copy.copy) == (two.phases is one.phases)
        for name in Rotary.__slots__:
            a, b = getattr(one, name), getattr(two, name)
            assert type(a) is type(b) and (torch.equal(a, b) if isinstance(a, torch.Tensor) else a == b), name
        with pytest.raises(AttributeError, match="made of"):
            two.pairs = 1 << 20


def test_rotary_of_other_parts_is_refused():
    phases = torch.arange(4)
    for parts in ((phases[:0], None, 1, False, 1.0), (phases.int(), None, 1, False, 1.0), (phases[::2], None, 1, False, 1.0),
                  (phases, phases[:3], 2, False, 1.0), (phases, None, 2, False, 1.0), (phases, phases, 65, False, 1.0),
                  (phases, None, 1, False, float("inf")), (phases[None], None, 1, False, 1.0)):
        with pytest.raises(ValueError, match="rotary"):
            _rotary_of(Rotary, *parts)


@pytest.mark.parametrize("made", COPIES, ids=lambda f: f.__name__)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float8_e4m3fn], ids=str)
def test_paged_cache(made, dtype):
    one = PagedCache.zeros(3, 16, 2, 64, dtype, device="cpu")
    one.values.view(torch.uint8).copy_(torch.randint(0, 100, (*one.values.view(torch.uint8).shape,)))
    if one.scales is not None:
        one.scales.uniform_()
    for two in (made(one), made(Holder(one)).thing):
        assert type(two) is PagedCache and two.values.dtype == dtype
        assert torch.equal(two.values.view(torch.uint8), one.values.view(torch.uint8))
        assert two.scales is None if one.scales is None else torch.equal(two.scales, one.scales)
        # A shallow copy is another view of the same pages, the others are pages of their own.
        assert (made is copy.copy) == (two.values.data_ptr() == one.values.data_ptr())
        with pytest.raises(AttributeError, match="made of"):
            two.values = one.values


@pytest.mark.parametrize("made", COPIES, ids=lambda f: f.__name__)
def test_request_adapters(made):
    g = torch.Generator().manual_seed(3)
    pack = [tuple(LowRankResidual(torch.randn((r, 32), generator=g), torch.randn((n, r), generator=g), 0.5) for n in (48, 16))
            for r in (3, 20)]
    one = stack_request_adapters(pack, 32, (48, 16), device="cpu")
    for two in (made(one), made(Holder(one)).thing):
        assert type(two) is RequestAdapters and two.widths == (48, 16) and list(two.c_widths) == [48, 16]
        for name in ("down", "up", "scaling", "ranks"):
            assert torch.equal(getattr(two, name), getattr(one, name))
            assert (made is copy.copy) == (getattr(two, name).data_ptr() == getattr(one, name).data_ptr())
