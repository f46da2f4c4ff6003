"""The language-model example with no blocks at all: an embedding, a norm and a head, as small as a run of it gets."""
import os
import sys

import pytest

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads", [0, 4])
def test_example_without_blocks_runs(heads):
    import train_language_model as example

    losses = example.train(3, 128, 0, 500, 256, heads=heads)
    assert len(losses) == 3 and all(0 < x < 20 for x in losses)
