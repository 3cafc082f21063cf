"""examples/mx4_experts.py: the operators run together as a model's training
step; the loss has to fall to well below where it started."""
import os
import sys

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "examples"))

pytestmark = pytest.mark.gpu


def test_training_on_mx4_lowers_the_loss():
    import mx4_experts

    losses = mx4_experts.train(steps=25)
    assert np.isfinite(losses).all()
    assert losses[-1] < 0.7 * losses[0], losses
