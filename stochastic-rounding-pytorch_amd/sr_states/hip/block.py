"""FP8 matrices with a scale for each block of 128, their product, and a linear layer on it.

A ``BlockScaled`` matrix holds FP8 values (rows, k), the contracted axis last,
and a scale for each block: one row (or 128 rows) by 128 values of the
contracted axis.  ``block_cast`` makes one with this package's rounding rules
and power-of-two scales, so that the rounding to FP8 is the only one.
``block_matmul`` multiplies two of them on gfx950's FP8 matrix instructions,
which apply power-of-two scales themselves; FP32 scales, as checkpoints hold
them, multiply each block's sum in FP32.  ``block_linear`` is a linear layer
whose three products (forward, input gradient, weight gradient) run that way,
with the gradient rounded stochastically by default.

The reference package has no counterpart.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from .. import _lib
from .._hash import state_key
from ..formats import StateFormat, resolve_formats
from ..rounding import native_codes
from ._common import validate_device
from ._optimizer import reject_dtensors

BLOCK = _lib.BLOCK
FP8_DTYPES = (torch.float8_e4m3fn, torch.float8_e5m2)
_WIDE_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_SCALE_TYPES = {torch.float8_e8m0fnu: _lib.SCALE_E8M0, torch.float32: _lib.SCALE_F32}


class BlockScaled(NamedTuple):
    """FP8 values and the scales of their blocks of 128.

    ``data``: (rows, k) FP8 with consecutive columns.  ``scale``: E8M0 or FP32,
    (rows, ceil(k / 128)) for blocks of one row, or (ceil(rows / 128),
    ceil(k / 128)) for blocks of 128 rows.  Value (r, c) is
    ``data[r, c] * scale[r or r // 128, c // 128]``.
    """

    data: torch.Tensor
    scale: torch.Tensor

    def dequantize(self) -> torch.Tensor:
        """The FP32 values the matrix stands for."""
        rows, k = self.data.shape
        scale = self.scale.float()
        if scale.shape[0] != rows:
            scale = scale.repeat_interleave(BLOCK, 0)[:rows]
        return self.data.float() * scale.repeat_interleave(BLOCK, 1)[:, :k]


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _row_stride(x: torch.Tensor, what: str) -> int:
    """The distance between rows of a 2-D tensor with consecutive columns."""
    rows, cols = x.shape
    stride = x.stride(0) if rows > 1 else max(cols, 1)
    if (cols > 1 and x.stride(1) != 1) or stride < cols:
        raise ValueError(f"{what} requires consecutive columns and rows that do not overlap")
    return stride


def _new_output(rows: int, k: int, dtype, square: bool, device):
    """An empty BlockScaled; rows start on 16 bytes, which the product's asynchronous loads need."""
    data = torch.empty_strided((rows, k), (-(-k // 16) * 16, 1), dtype=dtype, device=device)
    scale = torch.empty((_blocks(rows) if square else rows, _blocks(k)), dtype=torch.float8_e8m0fnu, device=device)
    return BlockScaled(data, scale)


def _address(x: torch.Tensor) -> int:
    return x.data_ptr()


def block_cast(
    x: torch.Tensor,
    *,
    dtype: torch.dtype = torch.float8_e4m3fn,
    block: tuple = (1, BLOCK),
    axis: int | tuple = 1,
    rounding: str = "stochastic",
    seed: int = 0,
    offset: int = 0,
):
    """Quantize a GPU matrix (rows, cols; FP32, BF16 or FP16) to FP8 with a scale for each block of 128.

    ``axis`` is the axis a product will contract: 1 gives blocks along the
    columns and data (rows, cols); 0 gives blocks along the rows and data
    (cols, rows), transposed; the tuple ``(1, 0)`` or ``(0, 1)`` gives both in
    its order from one pass over ``x``.  ``block`` is (1, 128) or (128, 128).

    A block's scale is the smallest power of two (E8M0, at least 2**-127) that
    brings its largest finite magnitude into the format's range, 1 for a
    block of zeros.  The scaled values are rounded as :func:`sr_states.cast`
    rounds them: element (r, c) uses counter ``r * cols + c + seed + offset``
    (mod 2**32) in either orientation, infinities saturate and NaN stays.

    The data's rows start on multiples of 16 bytes, so ``data`` is
    contiguous only where its last size is one.  Nothing is recorded for
    autograd.
    """
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"expected a tensor, got {type(x).__name__}")
    reject_dtensors(x)
    if x.dtype not in _WIDE_DTYPES:
        raise TypeError(f"expected FP32, BF16 or FP16 input, got {x.dtype}")
    if dtype not in FP8_DTYPES:
        raise ValueError(f"block casts give torch.float8_e4m3fn or torch.float8_e5m2, not {dtype}")
    code, rule = native_codes(dtype, rounding)
    block = tuple(block)
    if block not in ((1, BLOCK), (BLOCK, BLOCK)):
        raise ValueError(f"block must be (1, {BLOCK}) or ({BLOCK}, {BLOCK})")
    axes = axis if isinstance(axis, tuple) else (axis,)
    if axes not in ((1,), (0,), (1, 0), (0, 1)):
        raise ValueError("axis must be 1, 0, (1, 0) or (0, 1)")
    if x.dim() != 2:
        raise ValueError(f"block_cast takes a matrix, not {x.dim()} dimensions")
    device = x.device
    if device.type != "cuda":
        raise ValueError("block_cast requires a GPU tensor")
    validate_device(device)
    stride = _row_stride(x, "block_cast")
    rows, cols = x.shape
    square = block[0] == BLOCK
    result = {}
    out = {}
    for a in axes:
        q = _new_output(*((rows, cols) if a == 1 else (cols, rows)), dtype, square, device)
        result[a] = q
        out[a] = _lib.BlockOutput(_address(q.data), _address(q.scale), q.data.stride(0), max(q.scale.shape[1], 1))
    if rows and cols:
        with _lib.on_device(device):
            _lib.call(
                "sr_block_cast", _address(x), stride, rows, cols, _lib.DTYPE_CODES[x.dtype], code, rule, int(square),
                _lib.low32(seed), _lib.low32(offset), out.get(1), out.get(0), _lib.stream_handle(device),
            )
    return result[axes[0]] if len(axes) == 1 else tuple(result[a] for a in axes)


def _operand(q: BlockScaled, name: str) -> _lib.BlockMatrix:
    """The checked C record of one operand."""
    data, scale = q
    for t in (data, scale):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a BlockScaled pair of tensors")
    reject_dtensors(data, scale)
    if data.dtype not in FP8_DTYPES:
        raise TypeError(f"{name}: data must be FP8 (E4M3 or E5M2), got {data.dtype}")
    if scale.dtype not in _SCALE_TYPES:
        raise TypeError(f"{name}: scales must be torch.float8_e8m0fnu or torch.float32, got {scale.dtype}")
    if data.dim() != 2 or scale.dim() != 2:
        raise ValueError(f"{name}: data and scales must be matrices")
    if data.device.type != "cuda" or scale.device != data.device:
        raise ValueError(f"{name}: data and scales must be on the same GPU device")
    rows, k = data.shape
    if scale.shape[1] != _blocks(k) or scale.shape[0] not in (rows, _blocks(rows)):
        raise ValueError(
            f"{name}: scales of a {rows} x {k} matrix are {rows} x {_blocks(k)} or {_blocks(rows)} x {_blocks(k)}, "
            f"not {tuple(scale.shape)}"
        )
    return _lib.BlockMatrix(
        _address(data), _address(scale), _row_stride(data, f"{name}: data"), _row_stride(scale, f"{name}: scale"),
        rows, _lib.DTYPE_CODES[data.dtype], _SCALE_TYPES[scale.dtype], 1 if scale.shape[0] == rows else BLOCK, 0,
    )


def _span(x: torch.Tensor):
    """First and one past the last byte a 2-D tensor touches."""
    start = x.data_ptr()
    if not x.numel():
        return start, start
    last = sum((n - 1) * s for n, s in zip(x.shape, x.stride()))
    return start, start + (last + 1) * x.element_size()


def block_matmul(
    a: BlockScaled,
    b: BlockScaled,
    *,
    out_dtype: torch.dtype | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``a @ b.T`` of two block-scaled matrices (m, k) and (n, k), as an (m, n) tensor.

    Either may be E4M3 or E5M2 with blocks of one row or of 128; both have E8M0
    scales or both FP32 ones.  Products are summed in FP32 and rounded once, to
    ``out_dtype`` (BF16 by default, FP32 or FP16) or into ``out``, which has
    consecutive columns and shares no memory with the operands.
    """
    left, right = _operand(a, "a"), _operand(b, "b")
    device, k = a[0].device, a[0].shape[1]
    if b[0].device != device:
        raise ValueError("a and b must be on the same GPU device")
    if b[0].shape[1] != k:
        raise ValueError(f"a and b contract {k} and {b[0].shape[1]} values")
    if left.scale_type != right.scale_type:
        raise TypeError("a and b must have scales of one type")
    validate_device(device)
    m, n = left.rows, right.rows
    if out is None:
        dtype = torch.bfloat16 if out_dtype is None else out_dtype
        if dtype not in _WIDE_DTYPES:
            raise TypeError(f"out_dtype must be FP32, BF16 or FP16, not {dtype}")
        out = torch.empty((m, n), dtype=dtype, device=device)
        stride = n
    else:
        if out.dtype not in _WIDE_DTYPES or (out_dtype is not None and out.dtype != out_dtype):
            raise TypeError(f"out has dtype {out.dtype}")
        if out.shape != (m, n) or out.device != device:
            raise ValueError(f"out must be a {m} x {n} tensor on {device}")
        stride = _row_stride(out, "out")
        start, end = _span(out)
        for t in (*a, *b):
            first, last = _span(t)
            if start < last and first < end:
                raise ValueError("out must not overlap the operands")
    if m and n:
        size = _lib.library().sr_block_matmul_workspace(m, n, k)
        workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None
        with _lib.on_device(device):
            _lib.call(
                "sr_block_matmul", left, right, k, _address(out), stride, _lib.DTYPE_CODES[out.dtype],
                _address(workspace) if size else None, _lib.stream_handle(device),
            )
    return out


_LINEAR_NAMES = ("input", "weight", "gradient")
_LINEAR_FORMATS = (
    StateFormat(torch.float8_e4m3fn, "nearest"),
    StateFormat(torch.float8_e4m3fn, "nearest"),
    StateFormat(torch.float8_e4m3fn, "stochastic"),
)


def _matrix(x: torch.Tensor, cols: int) -> torch.Tensor:
    """x as rows of ``cols`` consecutive values, copied only where its layout needs it."""
    x = x.reshape(math.prod(x.shape[:-1]), cols)
    if (cols > 1 and x.stride(1) != 1) or (x.shape[0] > 1 and x.stride(0) < cols):
        x = x.contiguous()
    return x


class _BlockLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, formats, seed):
        rows = _matrix(x, weight.shape[1])
        need_x, need_w = ctx.needs_input_grad[:2]

        def cast(t, k, **options):
            fmt = formats[k]
            return block_cast(t, dtype=fmt.dtype, rounding=fmt.rounding, seed=state_key(seed, k), **options)

        ctx.cast, ctx.like, ctx.weight_dtype = cast, (x.shape, x.dtype), weight.dtype
        # The weight gradient contracts the tokens, so it needs the input's blocks along them; the input gradient
        # contracts the weight's rows, and its square blocks only turn.
        qx, qx_t = cast(rows, 0, axis=(1, 0)) if need_w else (cast(rows, 0), None)
        square = {"block": (BLOCK, BLOCK)}
        qw, qw_t = cast(_matrix(weight, weight.shape[1]), 1, axis=(1, 0), **square) if need_x else (
            cast(_matrix(weight, weight.shape[1]), 1, **square), None)
        ctx.save_for_backward(*(qx_t or (None, None)), *(qw_t or (None, None)))
        y = block_matmul(qx, qw, out_dtype=x.dtype)
        return y.view(*x.shape[:-1], weight.shape[0])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x_data, x_scale, w_data, w_scale = ctx.saved_tensors
        shape, dtype = ctx.like
        need_x, need_w = ctx.needs_input_grad[:2]
        rows = _matrix(dy, dy.shape[-1])
        axes = (1,) * need_x + (0,) * need_w
        q = ctx.cast(rows, 2, axis=axes if len(axes) > 1 else axes[0])
        q = dict(zip(axes, q if len(axes) > 1 else (q,)))
        dx = dw = None
        if need_x:
            dx = block_matmul(q[1], BlockScaled(w_data, w_scale), out_dtype=dtype).view(shape)
        if need_w:
            dw = block_matmul(q[0], BlockScaled(x_data, x_scale), out_dtype=ctx.weight_dtype)
        return dx, dw, None, None


def block_linear(
    x: torch.Tensor,
    weight: torch.Tensor,
    *,
    seed: int = 0,
    formats: StateFormat | dict | tuple | None = None,
) -> torch.Tensor:
    """``x @ weight.T`` with FP8 operands and block scales, forward and backward.

    ``x`` is (..., k) and ``weight`` (n, k), each FP32, BF16 or FP16 on the GPU;
    the result has x's dtype, the gradients their tensors' dtypes.  x and the
    gradient are quantized in blocks of one row by 128 contracted values, the
    weight in blocks of 128 by 128:

    - ``y  = Q(x) Q(weight)^T``
    - ``dx = Q(dy) Q(weight)``
    - ``dw = Q(dy)^T Q(x)``, both requantized with blocks along the tokens

    ``formats`` names the FP8 format and rule of "input", "weight" and
    "gradient" (one StateFormat for all, or a dict); by default E4M3,
    nearest for the first two and stochastic for the gradient.  Tensor k of
    that order uses the random stream ``state_key(seed, k)``, so ``seed`` should
    be an update key that differs by layer and step (:func:`sr_states.update_key`).
    Only the FP8 copies are kept for the backward pass.
    """
    chosen = _LINEAR_FORMATS if formats is None else resolve_formats(_LINEAR_NAMES, formats, backend="hip")
    for name, fmt in zip(_LINEAR_NAMES, chosen):
        if fmt.dtype not in FP8_DTYPES:
            raise ValueError(f"{name} format must be FP8, not {fmt.dtype}")
    for name, t in (("x", x), ("weight", weight)):
        reject_dtensors(t)
        if t.dtype not in _WIDE_DTYPES:
            raise TypeError(f"{name} must be FP32, BF16 or FP16, not {t.dtype}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x {tuple(x.shape)} and weight {tuple(weight.shape)} do not match")
    if x.device.type != "cuda" or weight.device != x.device:
        raise ValueError("x and weight must be on the same GPU device")
    return _BlockLinear.apply(x, weight, chosen, _lib.low32(seed))
