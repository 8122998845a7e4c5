"""examples/gated_delta_net.py: the layer operators together, trained and served.

Tolerances.  Served and trained outputs pass some 8 roundings to bf16 a block
(2^-9 each, independent), 2 blocks and the last norm: about 4.5 x 2^-9; 2^-5 leaves a
factor of 3.5 for what the blocks amplify.  Int8 codes put about 1% on a state (a
128-value row's largest is near 4 times its norm a value: 4 / 127 / sqrt(12)), and so on
each block's output; 2^-3 leaves the same factor.  A wrong state, slot or token is off
by its whole size."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = Path(__file__).resolve().parents[1] / "examples" / "gated_delta_net.py"
    spec = importlib.util.spec_from_file_location("gated_delta_net", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.fixture(scope="module")
def trained(example, device):
    torch.manual_seed(11)
    generator = torch.Generator().manual_seed(11)
    net = example.Net().to(device)
    return net, example.train(net, 60, device, generator)


def test_training_lowers_the_loss(trained):
    losses = trained[1]
    first, last = sum(losses[:5]) / 5, sum(losses[-5:]) / 5
    print(f"loss {first:.3f} -> {last:.3f}", flush=True)
    assert last < 0.9 * first


@pytest.mark.parametrize("lengths", [[64], [70, 1, 260, 33], [5, 129]])
def test_serving_gives_the_trained_outputs(example, trained, device, lengths):
    off = example.serve(trained[0], lengths, 20, device, torch.Generator().manual_seed(3))
    print(off, flush=True)
    assert off["decoded"] <= 2.0 ** -5
    assert off["decoded from int8 states"] <= 2.0 ** -3
    assert off["decoded by windowed int8 steps"] <= 2.0 ** -3
