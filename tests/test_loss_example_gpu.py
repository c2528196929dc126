"""The example that trains an engram with each loss in turn: every loss goes down, the pairs' margin and the sampled
answers' reward go up."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    spec = importlib.util.spec_from_file_location("train_engram_losses", os.path.join(ROOT, "examples", "train_engram_losses.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_every_loss_trains_the_engram():
    torch.manual_seed(0)
    kl, loss, margin, reward = _example().main(steps=30)
    assert kl[-1] < 0.5 * kl[0]
    assert loss[-1] < 0.5 * loss[0] and margin[-1] > margin[0] + 1.0
    assert sum(reward[-5:]) / 5 > reward[0] + 0.1
