"""examples/packed_moe_layer.py on the MI355X: weights packed by this package's encoder, run by
its products, and the router trained through them."""

import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(__file__), "..", "examples", "packed_moe_layer.py")


def test_packed_moe_layer(dev):
    spec = importlib.util.spec_from_file_location("packed_moe_layer", PATH)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    moe, one, losses = example.layer(train=8)
    # INT2 rows on a quarter of each tensor cost about a fifth of the product's norm (uniform
    # rounding to 4 levels of a unit normal leaves a relative error near 0.35 on those rows,
    # 16 levels 0.1): sqrt(.25 .35^2 + .75 .1^2) = 0.2; three products and the residual less
    assert 0.02 < one < 0.4 and 0.01 < moe < 0.6
    assert len(losses) == 8 and losses[-1] < losses[0]
