"""The predictor example end to end: layer norm, attention over scenes of
unequal length and the orthogonalised updates, trained through the rasterizer."""
import math

import pytest

pytestmark = pytest.mark.gpu


def test_training_lowers_the_loss(gpu):
    # untrained, the images are near the background: a loss of about 0.3, of which
    # 30 steps have to take more than a third
    from blitzgs_amd.examples import train_predictor
    losses = train_predictor.train(steps=30)
    assert all(math.isfinite(x) for x in losses)
    assert min(losses[-5:]) < 0.7 * losses[0], losses
