"""The sequence example runs in every form, and its served outputs are those of the
whole lists up to the cache's rounding."""

import sys
from pathlib import Path

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("positions", [False, True])
@pytest.mark.parametrize("bits", [16, 4])
def test_runs(dev, positions, bits):
    import sequence_model

    torch.manual_seed(0)
    model = sequence_model.SequenceModel(100, positions=50 if positions else 0)
    losses = sequence_model.train(model, 6, 40, 100, 2)
    assert len(losses) == 2 and all(map(torch.isfinite, torch.tensor(losses)))
    got, want = sequence_model.serve(model, 6, 40, 100, 3, bits)
    assert got.shape == want.shape and torch.isfinite(got.float()).all()
    off = float((got - want).float().norm() / want.float().norm())
    # 16 bits: the same rows, a few bf16 roundings.  4 bits: a row's values are off by
    # up to a thirtieth of its range (about four standard deviations), in keys and in values.
    assert off < (0.02 if bits == 16 else 0.3)
