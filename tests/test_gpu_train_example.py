"""examples/train_mace.py: the layer norms, their second order and the optimizer together.  The mean loss of the last
pass over the data is below half of the first's, with either kind of state."""

import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    spec = importlib.util.spec_from_file_location("train_mace", os.path.join(ROOT, "examples", "train_mace.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("bits", [32, 8])
def test_training_lowers_the_loss(bits):
    losses = _example().train(60, state_bits=bits)
    assert sum(losses[-4:]) < 0.5 * sum(losses[:4]), losses
