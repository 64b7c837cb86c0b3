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


class BlockScaled(NamedTuple):
    """FP8 values and the scales of their blocks of 128.

    ``data``: (rows, k) FP8 with consecutive columns.  ``scale``: E8M0 or FP32,
    (rows, ceil(k / 128)) for blocks of one row, or (ceil(rows / 128),
    ceil(k / 128)) for blocks of 128 rows.  Value (r, c) is
    ``data[r, c] * scale[r or r // 128, c // 128]``.  A stack of matrices has
    one more dimension in front of both.
    """

    data: torch.Tensor
    scale: torch.Tensor

    def dequantize(self) -> torch.Tensor:
        """The FP32 values the matrix stands for."""
        rows, k = self.data.shape[-2:]
        scale = self.scale.float()
        if scale.shape[-2] != rows:
            scale = scale.repeat_interleave(BLOCK, -2)[..., :rows, :]
        return self.data.float() * scale.repeat_interleave(BLOCK, -1)[..., :k]


# Checked (dtype, block, axis, rounding) of block_cast, as the native entry takes them: built-in rules
# can never be replaced, so what was checked once holds for the life of the process.
_CASTS: dict = {}


def _cast_plan(dtype, block, axis, rounding):
    if dtype not in FP8_DTYPES:
        raise ValueError(f"block casts give torch.float8_e4m3fn or torch.float8_e5m2, not {dtype}")
    code, rule = native_codes(dtype, rounding)
    block = tuple(block)
    if block not in ((1, BLOCK), (BLOCK, BLOCK)):
        raise ValueError(f"block must be (1, {BLOCK}) or ({BLOCK}, {BLOCK})")
    axes = axis if isinstance(axis, tuple) else (axis,)
    if axes not in ((1,), (0,), (1, 0), (0, 1)):
        raise ValueError("axis must be 1, 0, (1, 0) or (0, 1)")
    return code, rule, int(block[0] == BLOCK), "".join(str(int(a)) for a in axes)


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
    try:
        plan = _CASTS[dtype, block, axis, rounding]
    except KeyError:
        plan = _CASTS[dtype, block, axis, rounding] = _cast_plan(dtype, block, axis, rounding)
    except TypeError:  # an unhashable argument
        plan = _cast_plan(dtype, block, axis, rounding)
    device = _device_of(x)
    q = _lib.matrix().block_cast(x, *plan, seed & 0xFFFFFFFF, offset & 0xFFFFFFFF, _stream(device))
    if not isinstance(q, tuple):
        _lib.check("sr_block_cast", q)
    return BlockScaled(q[0], q[1]) if len(q) == 2 else (BlockScaled(q[0], q[1]), BlockScaled(q[2], q[3]))


def _device_of(*tensors):
    """The first tensor's device, checked where it is a GPU; the native entries refuse everything else."""
    reject_dtensors(*tensors)
    device = getattr(tensors[0], "device", None)
    if device is not None and device.type == "cuda":
        validate_device(device)
        return device
    return None


def _stream(device) -> int:
    return 0 if device is None else _lib.stream_handle(device)


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
    consecutive columns, shares no memory with the operands and, in grad mode,
    requires no gradient.  Nothing is recorded for autograd.
    """
    (a_data, a_scale), (b_data, b_scale) = a, b
    if out_dtype is None:
        code = -1  # out's, or BF16
    elif out_dtype in _WIDE_DTYPES:
        code = _lib.DTYPE_CODES[out_dtype]
    else:
        raise TypeError(f"out_dtype must be FP32, BF16 or FP16, not {out_dtype}")
    device = _device_of(a_data, a_scale, b_data, b_scale, out)
    result = _lib.matrix().block_matmul(a_data, a_scale, b_data, b_scale, code, out, _stream(device))
    if not isinstance(result, torch.Tensor):
        _lib.check("sr_block_matmul", result)
    return result


_LINEAR_NAMES = ("input", "weight", "gradient")
_LINEAR_FORMATS = (
    StateFormat(torch.float8_e4m3fn, "nearest"),
    StateFormat(torch.float8_e4m3fn, "nearest"),
    StateFormat(torch.float8_e4m3fn, "stochastic"),
)


# Checked formats of block_linear, as the native entries take them.
_LINEAR_CODES: dict = {}


def _linear_codes(formats):
    chosen = _LINEAR_FORMATS if formats is None else resolve_formats(_LINEAR_NAMES, formats, backend="hip")
    for name, fmt in zip(_LINEAR_NAMES, chosen):
        if fmt.dtype not in FP8_DTYPES:
            raise ValueError(f"{name} format must be FP8, not {fmt.dtype}")
    return tuple(code for fmt in chosen for code in native_codes(fmt.dtype, fmt.rounding))


def _formats_of(formats):
    try:
        return _LINEAR_CODES[formats]
    except KeyError:
        codes = _LINEAR_CODES[formats] = _linear_codes(formats)
        return codes
    except TypeError:  # a dict of formats
        return _linear_codes(formats)


class _BlockLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, codes, seed, recorded):
        # needs_input_grad says which tensors require gradients in every grad mode, and the mode is always off in here:
        # `recorded` is the caller's.
        need_x, need_w = (recorded and need for need in ctx.needs_input_grad[:2])
        seeds = tuple(state_key(seed, k) for k in range(3))
        # The weight gradient contracts the tokens, so it needs the input's blocks along them; the input gradient
        # contracts the weight's rows, and its square blocks only turn.
        out = _lib.matrix().linear_forward(x, weight, codes, seeds, need_x, need_w, _stream(x.device))
        if not isinstance(out, tuple):
            _lib.check("block_linear", out)
        ctx.save_for_backward(*out[1:])
        ctx.options = (*codes[4:], seeds[2], _lib.DTYPE_CODES[x.dtype], _lib.DTYPE_CODES[weight.dtype])
        return out[0]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        out = _lib.matrix().linear_backward(dy, *ctx.saved_tensors, *ctx.options, _stream(dy.device))
        if not isinstance(out, tuple):
            _lib.check("block_linear", out)
        return *out, None, None, None


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
    Only the FP8 copies are kept for the backward pass; without grad mode
    those that it alone would need are not made.
    """
    codes = _formats_of(formats)
    for name, t in (("x", x), ("weight", weight)):
        if t.dtype not in _WIDE_DTYPES:
            raise TypeError(f"{name} must be FP32, BF16 or FP16, not {t.dtype}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x {tuple(x.shape)} and weight {tuple(weight.shape)} do not match")
    if x.device.type != "cuda" or weight.device != x.device:
        raise ValueError("x and weight must be on the same GPU device")
    _device_of(x, weight)
    return _BlockLinear.apply(x, weight, codes, _lib.low32(seed), torch.is_grad_enabled())
