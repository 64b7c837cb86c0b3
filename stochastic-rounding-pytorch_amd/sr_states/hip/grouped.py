"""FP8 products whose rows are sorted into groups, each with a matrix of its own, and a linear layer on them.

The layers of a model of experts: rows (tokens) come sorted by expert, and
``sizes``, a tensor of the GPU, says how many rows each expert has.  No call
waits for the sizes, so a step with them can be captured into a graph and
replayed with others.  Everything else is as in :mod:`sr_states.hip.block`:
``grouped_block_cast`` quantizes, ``grouped_block_matmul`` multiplies each
group's rows by its own matrix, or contracts its own rows for the matrix's
gradient, and ``grouped_block_linear`` is the layer with its gradients.

The reference package has no counterpart.
"""

from __future__ import annotations

import torch

from .. import _lib
from .._hash import state_key
from ..formats import StateFormat
from .block import _CASTS, _WIDE_DTYPES, BLOCK, BlockScaled, _cast_plan, _device_of, _formats_of, _stream


def grouped_block_cast(
    x: torch.Tensor,
    sizes: torch.Tensor | None = None,
    *,
    dtype: torch.dtype = torch.float8_e4m3fn,
    block: tuple = (1, BLOCK),
    axis: int | tuple = 1,
    rounding: str = "stochastic",
    seed: int = 0,
    offset: int = 0,
):
    """:func:`block_cast` of a matrix whose rows are in groups, or of a stack of matrices.

    With ``sizes`` (int32 or int64, on the GPU; at most 4096 groups), ``x`` is
    (rows, cols) and group g its next ``sizes[g]`` rows; rows may remain behind
    the last group.  Axis 1 is :func:`block_cast`'s.  Axis 0 gives the transposed
    data (cols, columns) with blocks along each group's own rows: a group's
    columns start on the next multiple of 128 behind the group before, and
    zeros with a scale of 1 fill what belongs to no row.  ``columns`` is ``rows + 127
    * min(rows, groups)`` rounded down to a multiple of 128, room for any sizes.
    Blocks are (1, 128).

    Without ``sizes``, ``x`` is (matrices, rows, cols), and every matrix is cast
    by itself: data and scales have that dimension in front.

    Element i of ``x`` in memory order uses counter ``i + seed + offset`` (mod
    2**32) in either orientation.  Sizes below zero count as zero, and groups end
    where the rows do.  Nothing is recorded for autograd.
    """
    try:
        plan = _CASTS[dtype, block, axis, rounding]
    except KeyError:
        plan = _CASTS[dtype, block, axis, rounding] = _cast_plan(dtype, block, axis, rounding)
    except TypeError:  # an unhashable argument
        plan = _cast_plan(dtype, block, axis, rounding)
    device = _device_of(x) if sizes is None else _device_of(x, sizes)
    q = _lib.matrix().grouped_cast(x, sizes, *plan, seed & 0xFFFFFFFF, offset & 0xFFFFFFFF, _stream(device))
    if not isinstance(q, tuple):
        _lib.check("grouped_block_cast", q)
    return BlockScaled(q[0], q[1]) if len(q) == 2 else (BlockScaled(q[0], q[1]), BlockScaled(q[2], q[3]))


def grouped_block_matmul(
    a: BlockScaled,
    b: BlockScaled,
    sizes: torch.Tensor,
    *,
    out_dtype: torch.dtype | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Products of each group's rows with a matrix of its own, or with each other.

    Where ``b`` is a stack of matrices (groups, n, k) and ``a`` (m, k), the result is
    (m, n): ``a[t] @ b[g].T`` for the ``sizes[g]`` rows t of group g.  Rows behind the
    last group are zeros in a new result and keep what they hold in ``out``.

    Where ``b`` is a matrix (n, columns) and ``a`` (m, columns), the result is
    (groups, m, n): ``a[:, c] @ b[:, c].T`` over the columns c of group g, laid out
    as ``grouped_block_cast(axis=0)`` leaves them; zeros for a group without
    rows.  All columns of a group's blocks of 128 take part, and hold zeros
    behind its rows.

    Types, scales, ``out_dtype`` and ``out`` are those of :func:`block_matmul`;
    ``sizes`` is that of :func:`grouped_block_cast`.  Where 128 rows of ``a`` share a
    scale, they are counted from its first row, wherever groups start.
    """
    (a_data, a_scale), (b_data, b_scale) = a, b
    if out_dtype is None:
        code = -1  # out's, or BF16
    elif out_dtype in _WIDE_DTYPES:
        code = _lib.DTYPE_CODES[out_dtype]
    else:
        raise TypeError(f"out_dtype must be FP32, BF16 or FP16, not {out_dtype}")
    device = _device_of(a_data, a_scale, b_data, b_scale, sizes, out)
    result = _lib.matrix().grouped_matmul(a_data, a_scale, b_data, b_scale, sizes, code, out, _stream(device))
    if not isinstance(result, torch.Tensor):
        _lib.check("grouped_block_matmul", result)
    return result


def grouped_block_linear(
    x: torch.Tensor,
    weight: torch.Tensor,
    sizes: torch.Tensor,
    *,
    seed: int = 0,
    formats: StateFormat | dict | tuple | None = None,
) -> torch.Tensor:
    """:func:`block_linear` with a weight for each group of rows: ``x[t] @ weight[g].T``.

    ``x`` is (rows, k), ``weight`` (groups, n, k) and ``sizes`` (groups,) says how many
    rows each group has, in order (:func:`grouped_block_cast`); each of x and
    weight is FP32, BF16 or FP16 on the GPU.  The result (rows, n) has x's dtype,
    the gradients their tensors' dtypes.  Rows behind the last group give zeros
    and get a gradient of zero, and a group without rows gives its weight one.

    Quantization, ``formats``, ``seed`` and what is kept for the backward pass are
    :func:`block_linear`'s; the weights' blocks of 128 by 128 are those of each
    matrix, and the weight gradient's blocks along the tokens those of each
    group.  ``sizes`` must not change before the backward pass.
    """
    codes = _formats_of(formats)
    for name, t in (("x", x), ("weight", weight)):
        if t.dtype not in _WIDE_DTYPES:
            raise TypeError(f"{name} must be FP32, BF16 or FP16, not {t.dtype}")
    if weight.dim() != 3 or x.dim() != 2 or x.shape[1] != weight.shape[2]:
        raise ValueError(f"x {tuple(x.shape)} and weight {tuple(weight.shape)} do not match")
    if x.device.type != "cuda" or weight.device != x.device or sizes.device != x.device:
        raise ValueError("x, weight and sizes must be on the same GPU device")
    if sizes.shape != weight.shape[:1]:
        raise ValueError(f"{weight.shape[0]} weights take as many sizes, not {tuple(sizes.shape)}")
    device = _device_of(x, weight, sizes)
    key = _lib.low32(seed)
    y = _lib.matrix().grouped_linear(x, weight, sizes, codes, tuple(state_key(key, k) for k in range(3)), _stream(device))
    if not isinstance(y, torch.Tensor):
        _lib.check("grouped_block_linear", y)
    return y
