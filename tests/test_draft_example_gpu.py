"""The example's answers by trees of drafted tokens, for any number of answers.  Tolerance as
for the answers decoded token by token (tests/test_layer_example_gpu.py)."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("answers", [1, 2, 3, 9])
def test_any_number_of_answers(device, answers):
    path = Path(__file__).resolve().parents[1] / "examples" / "gated_delta_net.py"
    spec = importlib.util.spec_from_file_location("gated_delta_net", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    torch.manual_seed(5)
    net = example.Net().to(device)
    off = example.serve(net, [33, 1, 70], answers, device, torch.Generator().manual_seed(5))
    print(off, flush=True)
    assert off["decoded by trees"] <= 2.0 ** -5 and off["decoded"] <= 2.0 ** -5
