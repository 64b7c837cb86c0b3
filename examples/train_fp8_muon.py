"""Train a small regression network on FP8 block-scaled products with Muon and AdamW updates.

The hidden layers multiply in FP8 with a scale for each block of 128
(``block_linear``: activations and weights rounded to nearest, gradients
stochastically).  Muon updates their weights, which are matrices
(``orthogonalize`` inside, momentum in stochastically rounded BF16); AdamW
updates the rest.  After training, ``serve`` quantizes the weights once and
answers single rows with ``block_cast`` and ``block_matmul``.

    python examples/train_fp8_muon.py --steps 100
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "stochastic-rounding-pytorch_amd"))

import sr_states
import torch
from torch import nn

SEED = 7


class FP8Linear(nn.Linear):
    """A bias-free linear layer on ``block_linear``; ``key`` must differ by layer and step."""

    def __init__(self, inputs, outputs, **options):
        super().__init__(inputs, outputs, bias=False, **options)
        self.key = 0

    def forward(self, x):
        return sr_states.block_linear(x, self.weight, seed=self.key)


class Network(nn.Module):
    def __init__(self, width, depth, device):
        super().__init__()
        self.hidden = nn.ModuleList(FP8Linear(width, width, device=device) for _ in range(depth))
        self.gain = nn.Parameter(torch.ones(depth, width, device=device))
        self.head = nn.Linear(width, 1, device=device)

    def forward(self, x):
        for layer, gain in zip(self.hidden, self.gain):
            x = x + torch.relu(layer(x)) * gain
        return self.head(x)

    def start_step(self, step):
        """New random streams for this step's roundings."""
        for index, layer in enumerate(self.hidden):
            layer.key = sr_states.update_key(SEED, step, index)

    @torch.no_grad()
    def serve(self, rows):
        """The forward pass with weights quantized once; returns a function of a few rows."""
        weights = [sr_states.block_cast(layer.weight, block=(128, 128), rounding="nearest") for layer in self.hidden]

        def answer(x):
            with torch.no_grad():
                for weight, gain in zip(weights, self.gain):
                    y = sr_states.block_matmul(sr_states.block_cast(x, rounding="nearest"), weight, out_dtype=x.dtype)
                    x = x + torch.relu(y) * gain
                return self.head(x)

        return answer(rows)


def train(steps=100, width=256, depth=3, rows=512, device="cuda"):
    """Returns the trained network, its inputs and the loss of every step."""
    gen = torch.Generator(device=device).manual_seed(SEED)
    torch.manual_seed(SEED)
    x = torch.randn(rows, width, device=device, generator=gen)
    target = torch.tanh(x @ torch.randn(width, 1, device=device, generator=gen) / width**0.5)
    network = Network(width, depth, device)
    matrices = [layer.weight for layer in network.hidden]
    others = [network.gain, *network.head.parameters()]
    optimizers = [
        sr_states.MuonHip(matrices, lr=0.01, momentum=0.9, update_scale="rms", seed=SEED),
        sr_states.AdamWHip(others, lr=3e-3, seed=SEED),
    ]
    losses = []
    for step in range(steps):
        network.start_step(step)
        loss = (network(x) - target).square().mean()
        for optimizer in optimizers:
            optimizer.zero_grad()
        loss.backward()
        for optimizer in optimizers:
            optimizer.step()
        losses.append(float(loss.detach()))
    return network, x, losses


def main():
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=100)
    parser.add_argument("--width", type=int, default=256)
    arguments = parser.parse_args()
    network, x, losses = train(arguments.steps, arguments.width)
    for step in range(0, len(losses), max(1, len(losses) // 10)):
        print(f"step {step}: loss {losses[step]:.5f}")
    print(f"one row served: {float(network.serve(x[:1])):.4f}")


if __name__ == "__main__":
    main()
