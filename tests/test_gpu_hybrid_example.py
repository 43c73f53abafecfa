"""examples/hybrid_layer.py: both halves of a hybrid layer trained and served
together; the tokens served in pieces match one pass over the sequence."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "hybrid_layer.py")


def test_training_and_serving_agree():
    spec = importlib.util.spec_from_file_location("hybrid_layer", PATH)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    loss, grad, served, whole, cache = example.run()
    assert loss > 0 and torch.isfinite(grad).all() and grad.float().norm() > 0
    (sa, sr), (wa, wr) = (x.split([example.HQ * example.D, example.V_HEADS * example.D], -1) for x in (served, whole))
    # attention: o and the weights are rounded to bfloat16 on both sides, values up to
    # max |v|: 4 units of 2^-8 of the largest output
    assert (sa - wa).abs().max() <= 4 * 2.0 ** -8 * wa.abs().max()
    # the recurrence: the operator's stated output error on either side
    assert (sr - wr).abs().max() <= 2 * 2e-2 * wr.abs().max()
    held = len(cache.pages) - cache.pages.count(None)
    assert held <= -(-example.WINDOW // example.PAGE) + 2 + -(-example.SINKS // example.PAGE)
