"""Low-rank adapters of many requests at once, beside a projection that they share.

A batch's rows go through one projection (``block_linear``, or any other), and
each row adds the low-rank update of its own adapter: ``adapter_add``.  The
adapters of a batch are stacked, and ``index`` says which one each row uses, in
any order, or none.  The same call serves single tokens of many requests, a
prompt batch, and training, with gradients of the input and of the adapters.

The reference package has no counterpart.
"""

from __future__ import annotations

import torch

from .. import _lib
from .block import _device_of, _stream


def adapter_add(
    base: torch.Tensor,
    x: torch.Tensor,
    a: torch.Tensor,
    b: torch.Tensor,
    index: torch.Tensor,
    *,
    scaling: float | torch.Tensor = 1.0,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``base + scaling * (x @ a[i].T) @ b[i].T`` with an adapter ``i`` of its own for each row.

    ``x`` is (..., k) and ``base`` (..., n), the result of the projection that the
    rows share; ``a`` is (adapters, rank, k) and ``b`` (adapters, n, rank), rank 1
    to 128; all are FP32, BF16 or FP16, alike, on the GPU.  ``index`` (int32 or
    int64, x's shape without its last size) holds each row's adapter; a row
    whose number is outside [0, adapters) has none, and its result is ``base``'s.
    ``scaling`` is a number, or an FP32 tensor with one for each adapter, which
    gets no gradient.

    Sums are FP32 and the result is rounded once, at the end.  In BF16 calls a sum
    between two products (of x and a, and in the gradients of dy and b) enters
    the second to 2**-15 of itself, below the result's rounding unless the ranks
    cancel; infinities and NaN come out as the formula has them, for sums of
    2**-110 and more.

    Gradients flow to ``base``, ``x``, ``a`` and ``b``; adapters that no row uses get
    zeros.  ``x``, ``a``, ``b``, ``index`` and ``scaling`` are kept for the backward pass
    and must not change before it.  There are no forward-mode derivatives: an
    operand with a tangent is refused.  ``out``, which may be ``base`` itself, takes
    the result without recording gradients: in grad mode neither it nor an
    operand may require one.
    """
    device = _device_of(x, base, a, b, index, out)
    each = isinstance(scaling, torch.Tensor)
    if each:
        if scaling.requires_grad and torch.is_grad_enabled():
            raise ValueError("scaling gets no gradient: detach it")
        scale = 1.0
    else:
        scale, scaling = float(scaling), None
    result = _lib.matrix().adapter_add(base, x, a, b, index, scaling, scale, out, _stream(device))
    if not isinstance(result, torch.Tensor):
        _lib.check("adapter_add", result)
    return result
