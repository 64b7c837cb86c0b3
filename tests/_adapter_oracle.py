"""adapter_add and its gradients in 64 bits, adapter by adapter; any device.

Every result comes with the same sums over magnitudes, which bound its error.
"""

from __future__ import annotations

import torch


def _factor(scaling, i):
    return scaling if isinstance(scaling, float) else float(scaling[i])


def _rows(t):
    return t.detach().double().reshape(-1, t.shape[-1])


def add(base, x, a, b, index, scaling):
    base, x, index = _rows(base), _rows(x), index.reshape(-1)
    value, size = base.clone(), base.abs()
    for i in range(a.shape[0]):
        mine = (index == i).nonzero().flatten()
        low, high, s = a[i].detach().double().t().contiguous(), b[i].detach().double().t().contiguous(), _factor(scaling, i)
        value[mine] += s * (x[mine] @ low) @ high
        size[mine] += abs(s) * (x[mine].abs() @ low.abs()) @ high.abs()
    return value, size


def gradients(dy, x, a, b, index, scaling):
    """((dx, sizes), (da, sizes), (db, sizes))."""
    dy, x, index = _rows(dy), _rows(x), index.reshape(-1)
    out = [torch.zeros((2, *t.shape), dtype=torch.float64, device=x.device) for t in (x, a, b)]
    for i in range(a.shape[0]):
        mine = (index == i).nonzero().flatten()
        s = _factor(scaling, i)
        for part, f in ((0, lambda t: t), (1, torch.abs)):
            rows, grad, low, high = f(x[mine]), f(dy[mine]), f(a[i].detach().double()), f(b[i].detach().double())
            g, h = abs(s) * grad @ high, abs(s) * rows @ low.t().contiguous()
            if part == 0:
                g, h = g * (1 if s >= 0 else -1), h * (1 if s >= 0 else -1)
            out[0][part][mine] = g @ low
            out[1][part][i] = g.t().contiguous() @ rows
            out[2][part][i] = grad.t().contiguous() @ h
    return [(t[0], t[1]) for t in out]
