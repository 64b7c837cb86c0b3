"""Train a small mixture of experts on FP8 products, then adapters of it for several tasks at once.

Every block has a projection that all rows share (``block_linear``) and a layer
of experts: a router sends each row to one of them, the rows are sorted by
expert, and ``grouped_block_linear`` multiplies each group by its own weights
in FP8 with a scale for each block of 128.  AdamW updates the weights with
stochastically rounded BF16 moments.  Then the network stays as it is, and a
low-rank adapter for each task, added to the shared projections by
``adapter_add``, learns from batches that mix the tasks' rows.  ``serve``
answers rows of any tasks together.

    python examples/train_fp8_experts.py --steps 100
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


class Experts(nn.Module):
    """Two matrices for each of ``count`` experts, and the router that picks one of them for each row."""

    def __init__(self, width, hidden, count, device):
        super().__init__()
        self.router = nn.Linear(width, count, bias=False, device=device)
        self.up = nn.Parameter(torch.randn(count, hidden, width, device=device) * width**-0.5)
        self.down = nn.Parameter(torch.randn(count, width, hidden, device=device) * hidden**-0.5)

    def forward(self, x, key):
        weight, expert = torch.softmax(self.router(x), -1).max(-1)
        order = torch.argsort(expert, stable=True)
        # The sizes stay on the GPU: no call waits for them.
        sizes = torch.zeros(self.up.shape[0], dtype=torch.int64, device=x.device).scatter_add_(0, expert, torch.ones_like(expert))
        h = sr_states.grouped_block_linear(x[order], self.up, sizes, seed=sr_states.state_key(key, 0))
        h = sr_states.grouped_block_linear(torch.relu(h), self.down, sizes, seed=sr_states.state_key(key, 1))
        return torch.zeros_like(x).index_copy(0, order, h) * weight[:, None]


class Adapters(nn.Module):
    """A low-rank update of a square projection for each task; no effect before they are trained."""

    def __init__(self, width, rank, tasks, device):
        super().__init__()
        self.a = nn.Parameter(torch.randn(tasks, rank, width, device=device) * width**-0.5)
        self.b = nn.Parameter(torch.zeros(tasks, width, rank, device=device))


class Network(nn.Module):
    def __init__(self, width, depth, experts, device):
        super().__init__()
        self.shared = nn.ParameterList(nn.Parameter(torch.randn(width, width, device=device) * width**-0.5) for _ in range(depth))
        self.experts = nn.ModuleList(Experts(width, 2 * width, experts, device) for _ in range(depth))
        self.head = nn.Linear(width, 1, device=device)

    def forward(self, x, step=0, adapters=None, task=None):
        for index, (weight, experts) in enumerate(zip(self.shared, self.experts)):
            key = sr_states.update_key(SEED, step, index)  # this layer's and step's random streams
            y = sr_states.block_linear(x, weight, seed=sr_states.state_key(key, 2))
            if adapters is not None:
                y = sr_states.adapter_add(y, x, adapters[index].a, adapters[index].b, task, scaling=2.0)
            x = x + torch.relu(y)
            x = x + experts(x, key)
        return self.head(x)


def fit(network, parameters, x, target, steps, **options):
    """AdamW on ``parameters``; returns the loss of every step."""
    optimizer = sr_states.AdamWHip(parameters, lr=3e-3, seed=SEED)
    losses = []
    for step in range(steps):
        loss = (network(x, step, **options) - target).square().mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(float(loss.detach()))
    return losses


def train(steps=100, width=128, depth=2, experts=4, tasks=3, rows=512, device="cuda"):
    """Returns the trained network, its adapters, the inputs with their tasks, and both losses of every step."""
    gen = torch.Generator(device=device).manual_seed(SEED)
    torch.manual_seed(SEED)
    x = torch.randn(rows, width, device=device, generator=gen)
    goal = torch.randn(width, 1 + tasks, device=device, generator=gen) / width**0.5
    network = Network(width, depth, experts, device)
    losses = fit(network, list(network.parameters()), x, torch.tanh(x @ goal[:, :1]), steps)
    for parameter in network.parameters():
        parameter.requires_grad_(False)
    task = torch.randint(-1, tasks, (rows,), device=device, generator=gen)  # -1: the network as it is
    adapters = nn.ModuleList(Adapters(width, 8, tasks, device) for _ in range(depth))
    target = torch.tanh((x @ goal).gather(1, 1 + task[:, None]))
    adapted = fit(network, list(adapters.parameters()), x, target, steps, adapters=adapters, task=task)
    return network, adapters, x, task, losses, adapted


@torch.no_grad()
def serve(network, adapters, rows, task):
    """The answers to rows of any tasks."""
    return network(rows, adapters=adapters, task=task)


def main():
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=100)
    parser.add_argument("--width", type=int, default=128)
    arguments = parser.parse_args()
    network, adapters, x, task, losses, adapted = train(arguments.steps, arguments.width)
    for name, values in (("network", losses), ("adapters", adapted)):
        for step in range(0, len(values), max(1, len(values) // 5)):
            print(f"{name}, step {step}: loss {values[step]:.5f}")
    print("four rows served:", [round(float(v), 4) for v in serve(network, adapters, x[:4], task[:4]).flatten()])


if __name__ == "__main__":
    main()
