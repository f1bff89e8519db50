"""The example's training step: the operators together, from the embedding to Muon."""
import importlib.util
from pathlib import Path

import pytest


@pytest.mark.gpu
def test_example_learns(gpu):
    path = Path(__file__).resolve().parent.parent / "examples" / "train_step.py"
    spec = importlib.util.spec_from_file_location("train_step", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses = example.main(steps=30, batch=8, length=64, vocab=301, dim=128, verbose=False)
    assert all(a == a and b == b for a, b in losses)
    # log(301) = 5.7 and more before the first step; the teacher's own entropy is 1.7
    assert losses[0][0] > 5.0 and losses[-1][0] < 0.7 * losses[0][0]
    assert losses[-1][1] < 0.6 * losses[0][1]
