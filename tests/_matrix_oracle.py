"""64-bit forms of the matrix operators, written from their definitions; any device."""

from __future__ import annotations

import torch

BLOCK = 128
FORMATS = {  # dtype: (mantissa bits, smallest normal exponent, exponent of the maximum 1.75 * 2^top)
    torch.float8_e4m3fn: (3, -6, 8),
    torch.float8_e5m2: (2, -14, 15),
}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def h32(x):
    x = x & 0xFFFFFFFF
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def power(e):
    """2^e in float64, exactly (torch.ldexp takes the device's pow, which is not)."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def exponents(blocks, dtype):
    """The smallest e >= -127 with max|finite| <= 2^e * maximum for the last axis; 0 for zeros."""
    top = FORMATS[dtype][2]
    amax = torch.where(blocks.isfinite(), blocks.abs(), 0.0).amax(-1)
    mantissa, exponent = torch.frexp(amax)  # amax = mantissa * 2^exponent, 0.5 <= mantissa < 1
    e = exponent - 1 - top + (mantissa > 0.875)
    return torch.where(amax > 0, e, torch.zeros_like(e)).clamp(min=-127)


def block_cast(x, dtype, rule, square, axis, seed):
    """(values of the data, scales) as float64, in the orientation of `axis`."""
    mantissa, lowest, top = FORMATS[dtype]
    x = x.double()
    index = torch.arange(x.numel(), device=x.device).view(x.shape)
    if axis == 0:
        x, index = x.t().contiguous(), index.t()
    rows, cols = x.shape
    rb, cb = -(-rows // BLOCK), -(-cols // BLOCK)
    padded = torch.zeros(rb * BLOCK, cb * BLOCK, dtype=torch.float64, device=x.device)
    padded[:rows, :cols] = x
    tiles = padded.view(rb, BLOCK, cb, BLOCK).transpose(1, 2)
    if square:
        e = exponents(tiles.reshape(rb, cb, -1), dtype)
        per_row = e.repeat_interleave(BLOCK, 0)[:rows]
    else:
        e = per_row = exponents(padded.view(rb * BLOCK, cb, BLOCK), dtype)[:rows]
    y = x * power(-per_row.repeat_interleave(BLOCK, 1)[:, :cols])
    magnitude = y.abs().clamp(max=1.75 * 2.0**top)
    _, exponent = torch.frexp(magnitude)
    spacing = power((exponent - 1).clamp(min=lowest) - mantissa)
    steps = magnitude / spacing
    below = steps.floor()
    if rule == "nearest":
        result = steps.round()
    else:
        result = below + ((h32(index + seed) >> 8).double() < ((steps - below) * 2**24).floor())
    value = torch.where(y.isnan(), y, torch.copysign(result * spacing, y))
    return value, power(e)


def dequantize(data, scale):
    rows, cols = data.shape
    scale = scale.double()
    if scale.shape[0] != rows:
        scale = scale.repeat_interleave(BLOCK, 0)[:rows]
    return data.double() * scale.repeat_interleave(BLOCK, 1)[:, :cols]


def product(a, b):
    """(a b^T, the same of the magnitudes) of two (data, scale) pairs."""
    x, y = dequantize(*a), dequantize(*b)
    return x @ y.t().contiguous(), x.abs() @ y.abs().t().contiguous()


def orthogonalize(x, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    a, b, c = coefficients
    x = x.double()
    if x.shape[-2] > x.shape[-1]:
        return orthogonalize(x.mT.contiguous(), steps, coefficients, eps).mT.contiguous()
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    for _ in range(steps):
        gram = x @ x.mT.contiguous()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x


def relative(actual, expected):
    """The 2-norm of the difference over that of `expected` (or of the difference itself where that is 0)."""
    expected = expected.double()
    norm = expected.norm()
    off = (actual.double() - expected).norm()
    return float(off / norm if norm > 0 else off)
