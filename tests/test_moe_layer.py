"""The example layer: router, exchange and experts together, in two weight formats."""
import os
import sys

import pytest

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 50])
def test_both_formats_agree(tokens):
    """E2M1 weights in blocks of 32 keep a cosine of 0.99 to the values they stand
    for (relative error 0.12 a weight, of three products in a row), E4M3 0.999."""
    import moe_layer
    cosine, _ = moe_layer.run(tokens=tokens, hidden=512, inter=256, experts=16, topk=4, steps=2)
    assert cosine > 0.97
