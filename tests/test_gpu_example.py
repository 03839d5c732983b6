"""The example that runs the weight-only projections and packed attention together."""

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
EXAMPLE = Path(__file__).resolve().parents[1] / "examples" / "nvfp4_attention.py"


def test_growing_sequences_agree_with_whole_ones(dev):
    spec = importlib.util.spec_from_file_location("nvfp4_attention_example", EXAMPLE)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    grown, whole = example.run(dev)
    assert grown.shape == whole.shape == (3, 512) and bool(torch.isfinite(grown).all())
    # Both sides round the projection, the attention weights and output and the result to bf16, each
    # by half a step (2^-8 of the value) at most; the two differ where a sum's order moves a rounding
    # by a whole step.  Errors of single values add up as norms.
    assert (grown - whole).double().norm() <= 4 * 2.0**-7 * whole.double().norm()
