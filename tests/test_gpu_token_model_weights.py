"""The example model (examples/token_model.py) that trains on after its output matrix was quantised."""
import os
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "project-currennt-public_b200", "examples"))


@pytest.mark.parametrize("how", ["step", "learn"])
def test_the_8_bit_matrix_follows_the_weights(how):
    """a step between quantize() and last_logits() gives the logits of the new weights: the bits of a matrix that is quantised afresh"""
    import torch
    import token_model as tm
    model, g = tm.TokenModel(30, 40, 1, 6, 8, seed=3), torch.Generator().manual_seed(2)
    tokens, targets = tm.batch(6, 8, 30, g)
    model.quantize()
    if how == "step":
        model.step(tokens, targets, 0.5, 1.0)
    else:
        model.learn(tm.TokenModel(30, 48, 1, 6, 8, seed=9), tokens, 0.5, 1.0)
    model.load(tokens[:3].clamp(min=0))
    got = model.last_logits().clone()
    model.quantize()
    assert torch.equal(got, model.last_logits())
    model.synchronize()
