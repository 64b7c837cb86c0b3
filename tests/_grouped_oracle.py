"""64-bit forms of the grouped matrix operators, group by group from those of single matrices; any device."""

from __future__ import annotations

import _matrix_oracle as oracle
import torch

BLOCK = oracle.BLOCK


def counts_of(sizes, rows):
    """The groups' rows as a call takes them: none below zero, none beyond the matrix."""
    counts = []
    for n in sizes:
        counts.append(min(max(int(n), 0), rows - sum(counts)))
    return counts


def columns(rows, groups):
    return (rows + (BLOCK - 1) * min(rows, groups)) // BLOCK * BLOCK if groups else 0


def starts(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + -(-n // BLOCK) * BLOCK)
    return out[:-1]


def cast_columns(x, counts, dtype, rule, seed):
    """(values, scales) of the transposed cast with blocks along each group's rows."""
    width = columns(x.shape[0], len(counts))
    values = torch.zeros(x.shape[1], width, dtype=torch.float64, device=x.device)
    scales = torch.ones(x.shape[1], width // BLOCK, dtype=torch.float64, device=x.device)
    row = 0
    for at, n in zip(starts(counts), counts):
        if n:
            value, scale = oracle.block_cast(x[row:row + n], dtype, rule, False, 0, seed + row * x.shape[1])
            values[:, at:at + n] = value
            scales[:, at // BLOCK:at // BLOCK + scale.shape[1]] = scale
        row += n
    return values, scales


def cast_stack(x, dtype, rule, square, axis, seed):
    each = [oracle.block_cast(m, dtype, rule, square, axis, seed + i * m.numel()) for i, m in enumerate(x)]
    return torch.stack([v for v, _ in each]), torch.stack([s for _, s in each])


def product(a, b, counts):
    """(a[t] b[g]^T for the rows t of group g, the same of the magnitudes); zeros behind the last group."""
    n = b[0].shape[1]
    out = torch.zeros(2, a[0].shape[0], n, dtype=torch.float64, device=a[0].device)
    row = 0
    for g, count in enumerate(counts):
        if count:
            rows = (a[0][row:row + count], _rows_of(a, row, count))
            out[0, row:row + count], out[1, row:row + count] = oracle.product(rows, (b[0][g], b[1][g]))
        row += count
    return out[0], out[1]


def _rows_of(a, row, count):
    data, scale = a
    if scale.shape[0] != data.shape[0]:  # blocks of 128 rows
        scale = scale.repeat_interleave(BLOCK, 0)[:data.shape[0]]
    return scale[row:row + count]


def contract(a, b, counts):
    """(a[:, c] b[:, c]^T over the columns c of each group, the same of the magnitudes)."""
    out = torch.zeros(2, len(counts), a[0].shape[0], b[0].shape[0], dtype=torch.float64, device=a[0].device)
    for g, (at, n) in enumerate(zip(starts(counts), counts)):
        if n:
            width = -(-n // BLOCK) * BLOCK
            part = [(m[0][:, at:at + width], m[1][:, at // BLOCK:(at + width) // BLOCK]) for m in (a, b)]
            out[0, g], out[1, g] = oracle.product(*part)
    return out[0], out[1]
