"""The training example: FP8 products, Muon and AdamW together, then serving."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


def _example():
    path = Path(__file__).resolve().parent.parent / "examples" / "train_fp8_muon.py"
    spec = importlib.util.spec_from_file_location("train_fp8_muon", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_example_trains_and_serves(cuda):
    example = _example()
    network, x, losses = example.train(steps=40, device=cuda)
    assert losses[-1] < 0.5 * losses[0]
    # Rows are quantized by themselves, so one row's answer is the batch's, up to the few FP8 values of a layer (within
    # 2^-3 of each) that FP32 sums in another order tip to a neighbour.
    with torch.no_grad():
        batch = network(x[:20])
    one = network.serve(x[:1])
    torch.testing.assert_close(one, batch[:1], rtol=0, atol=0.05 * float(batch.abs().max()))

