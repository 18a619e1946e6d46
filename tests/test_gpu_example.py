"""The example model: the operators together, in training and in generation."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "sequence_model.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("sequence_model", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_training_learns(dev, example):
    torch.manual_seed(0)
    losses = example.train(example.Model().to(dev), 30)
    assert all(x == x for x in losses)
    # log 64 = 4.16 at first; the rule alone is worth 0.9 log(1 / 0.9) + 0.1 log(64 / 0.1) = 0.74
    assert losses[0] > 4 and losses[-1] < 2


def test_generation_continues_the_prompt(dev, example):
    """Token by token the logits are those of the whole sequence, up to bf16 roundings of
    four blocks: each rounds the residual once, 2^-8 of it at most, and computes from rounded values."""
    torch.manual_seed(0)
    model = example.Model().to(dev)
    example.train(model, 5)
    prompts = example.sequences(3, 90, 64, dev, torch.Generator().manual_seed(3))
    lengths = torch.tensor([90, 41, 1], dtype=torch.int32, device=dev)
    tokens, logits = model.generate(prompts, lengths, 12)
    for b, n in enumerate(lengths.tolist()):
        whole = torch.cat([prompts[b, :n], tokens[b]])[None]
        with torch.no_grad():
            want = model(whole)[0, n - 1:n + 11]
        assert (logits[b] - want).norm() < 8 * 2.0 ** -8 * want.norm()
