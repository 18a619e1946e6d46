"""What the example model cannot generate it refuses before any operator runs: no GPU is needed."""
import importlib.util
import os

import pytest
import torch

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "sequence_model.py")


@pytest.fixture(scope="module")
def model():
    spec = importlib.util.spec_from_file_location("sequence_model", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module.Model(length=32)


@pytest.mark.parametrize("width,lengths,n,what", [(20, [20, 4], 14, "32"), (20, [20, 0], 4, "empty"), (20, [20, 21], 4, "20"),
                                                  (33, [5, 5], 1, "32"), (20, [20, -1], 4, "empty")])
def test_generation_beyond_what_the_blocks_keep(model, width, lengths, n, what):
    """The convolution keeps `length` tokens: a position past them would be written outside."""
    with pytest.raises(ValueError, match=what):
        model.generate(torch.zeros(2, width, dtype=torch.long), torch.tensor(lengths, dtype=torch.int32), n)


def test_sequences_longer_than_the_filters(model):
    with pytest.raises(ValueError, match="32"):
        model(torch.zeros(2, 33, dtype=torch.long))
