"""GPU: table convolutions, the exact dense head, its cross entropy and AdamW in one training loop (examples/retrain_classifier.py)."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_network_learns(built, bits):
    spec = importlib.util.spec_from_file_location("retrain_classifier", os.path.join(ROOT, "examples", "retrain_classifier.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, right = example.train(steps=60, batch=128, state_bits=bits)
    # ten classes: 2.3 at the start, and far below when they are told apart
    assert 1.5 < losses[0] < 4.0 and sum(losses[-5:]) / 5 < 0.5 * losses[0] and right > 0.5
