"""The grouped operators' C ABI checks, refusals without a GPU, and their oracle (CPU)."""

from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import _grouped_oracle as grouped
import _matrix_oracle as oracle
import pytest
import sr_states
import torch
from sr_states import _lib

HEADER = Path(__file__).resolve().parents[1] / "include" / "sr_matrix_hip.h"


def test_structures_and_constants_match_the_header(tmp_path):
    source = tmp_path / "sizes.c"
    source.write_text(
        f'#include "{HEADER}"\n#include <stdio.h>\n'
        'int main(void) { printf("%zu %zu %d", sizeof(sr_groups), sizeof(sr_block_stack), SR_MATRIX_GROUPS); return 0; }\n'
    )
    program = tmp_path / "sizes"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", str(source), "-o", str(program)], check=True)
    sizes = [int(n) for n in subprocess.run([str(program)], capture_output=True, text=True, check=True).stdout.split()]
    assert sizes == [ctypes.sizeof(_lib.Groups), ctypes.sizeof(_lib.BlockStack), _lib.MATRIX_GROUPS]


@pytest.mark.parametrize("rows, groups", [(0, 3), (1, 1), (1, 5), (128, 1), (129, 2), (8192, 16), (100, 0), (7, 4096)])
def test_columns_have_room_for_any_sizes(rows, groups):
    width = _lib.library().sr_grouped_columns(rows, groups)
    assert width == grouped.columns(rows, groups) and width % 128 == 0
    if groups and rows:
        used = min(rows, groups)  # one row each, the rest in the last: the most blocks that can be
        counts = [1] * (used - 1) + [rows - used + 1]
        assert sum(-(-n // 128) * 128 for n in counts) <= width


def _matrix(**changes):
    fields = {"data": 1 << 20, "scale": 1 << 20, "ld": 128, "ld_scale": 1, "rows": 4, "dtype": _lib.SR_E4M3,
              "scale_type": 0, "block_rows": 1, **changes}
    return _lib.BlockMatrix(**fields)


def test_invalid_arguments_fail_before_any_device_work():
    lib = _lib.library()
    good, groups = _matrix(), _lib.Groups(1 << 20, 2, 0)

    def matmul(a=good, b=good, stride=512, k=128, g=groups, out=1 << 20, ldo=4, dtype=_lib.SR_BF16):
        return lib.sr_grouped_block_matmul(a, b, stride, 4, k, g, out, ldo, dtype, 1, None)

    def contract(a=good, b=good, columns=128, g=groups, out=1 << 20, ldo=4, stride=16, dtype=_lib.SR_BF16):
        return lib.sr_grouped_block_contract(a, b, columns, g, out, ldo, stride, dtype, None)

    wanted = _lib.BlockOutput(1 << 20, 1 << 20, 256, 2)

    def cast(x=1 << 20, rows=4, cols=256, x_dtype=0, dtype=_lib.SR_E4M3, rule=1, g=groups, by_rows=None, by_cols=wanted):
        return lib.sr_grouped_block_cast(x, 256, rows, cols, x_dtype, dtype, rule, 0, 0, g, by_rows, by_cols, None)

    stack = _lib.BlockStack(wanted, 1024, 8)

    def stacked(x=1 << 20, ldx=256, count=2, rows=4, cols=256, rule=1, by_rows=stack, by_cols=None):
        return lib.sr_stacked_block_cast(x, 1024, ldx, count, rows, cols, 0, _lib.SR_E4M3, rule, 0, 0, 0, by_rows, by_cols, None)

    too_many = _lib.Groups(1 << 20, 4097, 0)
    for call, message in [
        (lambda: matmul(a=_matrix(dtype=_lib.SR_BF16)), b"E4M3 or E5M2"),
        (lambda: matmul(b=_matrix(ld=100)), b"bytes between rows"),
        (lambda: matmul(b=_matrix(scale_type=1)), b"different scale types"),
        (lambda: matmul(g=None), b"null argument"),
        (lambda: matmul(g=too_many), b"4097 groups"),
        (lambda: matmul(g=_lib.Groups(1 << 20, -1, 0)), b"-1 groups"),
        (lambda: matmul(g=_lib.Groups(None, 2, 0)), b"null pointer"),
        (lambda: matmul(stride=-1), b"negative strides"),
        (lambda: matmul(k=-1), b"contracted"),
        (lambda: matmul(dtype=_lib.SR_E4M3), b"FP32, BF16 or FP16"),
        (lambda: matmul(out=None), b"null pointer"),
        (lambda: matmul(ldo=3), b"overlap"),
        (lambda: contract(columns=100), b"100 columns"),
        (lambda: contract(a=_matrix(data=(1 << 20) + 8)), b"16 bytes"),
        (lambda: contract(b=_matrix(ld=136)), b"16 bytes"),
        (lambda: contract(stride=15), b"overlap"),
        (lambda: contract(ldo=3), b"overlap"),
        (lambda: contract(out=None), b"null pointer"),
        (lambda: cast(x_dtype=_lib.SR_E4M3), b"FP32, BF16 or FP16"),
        (lambda: cast(dtype=_lib.SR_F16), b"E4M3 or E5M2"),
        (lambda: cast(rule=2), b"rounding rule"),
        (lambda: cast(g=too_many), b"4097 groups"),
        (lambda: cast(by_rows=wanted, by_cols=None), b"no output along"),
        (lambda: cast(by_cols=_lib.BlockOutput(1 << 20, 1 << 20, 255, 2)), b"overlap"),
        (lambda: cast(x=None), b"null pointer"),
        (lambda: stacked(count=-1), b"-1 matrices"),
        (lambda: stacked(count=4097), b"4097 matrices"),
        (lambda: stacked(ldx=255), b"overlap"),
        (lambda: stacked(rule=2), b"rounding rule"),
        (lambda: stacked(by_rows=None), b"no output"),
        (lambda: stacked(x=None), b"null pointer"),
    ]:
        assert call() == 1
        assert message in lib.sr_last_error()
    assert matmul(a=_matrix(rows=0, data=None, scale=None)) == 0  # empty: nothing to do
    assert contract(g=_lib.Groups(None, 0, 0)) == 0
    assert cast(rows=0) == 0 and stacked(count=0) == 0


def test_operators_refuse_cpu_tensors():
    x, w, sizes = torch.zeros(4, 256), torch.zeros(2, 8, 256), torch.tensor([1, 3], dtype=torch.int32)
    q = sr_states.BlockScaled(x.to(torch.float8_e4m3fn), torch.ones(4, 2))
    b = sr_states.BlockScaled(w.to(torch.float8_e4m3fn), torch.ones(2, 8, 2))
    for call in (lambda: sr_states.grouped_block_cast(x, sizes, axis=0), lambda: sr_states.grouped_block_cast(w),
                 lambda: sr_states.grouped_block_matmul(q, b, sizes), lambda: sr_states.grouped_block_linear(x, w, sizes)):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_public_names():
    for name in ("grouped_block_cast", "grouped_block_matmul", "grouped_block_linear"):
        assert name in sr_states.__all__ and name in sr_states.hip.__all__


def test_a_stack_dequantizes_matrix_by_matrix():
    data = torch.ones(2, 130, 200).to(torch.float8_e5m2)
    square = sr_states.BlockScaled(data, torch.arange(8.0).view(2, 2, 2)).dequantize()
    assert square.shape == (2, 130, 200) and square[1, 127, 0] == 4 and square[1, 128, 128] == 7
    rows = sr_states.BlockScaled(data, torch.arange(520.0).view(2, 130, 2)).dequantize()
    assert rows[1, 3, 127] == 266 and rows[1, 3, 128] == 267


def test_the_oracle_of_one_group_is_that_of_a_matrix():
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(256, 300, generator=gen)
    for rule in ("nearest", "stochastic"):
        values, scales = grouped.cast_columns(x, [256], torch.float8_e4m3fn, rule, 9)
        want = oracle.block_cast(x, torch.float8_e4m3fn, rule, False, 0, 9)
        assert torch.equal(values[:, :256], want[0]) and torch.equal(scales[:, :2], want[1])
    w = grouped.cast_stack(torch.randn(1, 20, 300, generator=gen), torch.float8_e4m3fn, "nearest", True, 1, 0)
    a = oracle.block_cast(x, torch.float8_e4m3fn, "nearest", False, 1, 0)
    assert torch.equal(grouped.product(a, w, [256])[0], oracle.product(a, (w[0][0], w[1][0]))[0])
    assert torch.equal(grouped.contract((values, scales), (values, scales), [256])[0][0], values.double().mul(
        scales.repeat_interleave(128, 1)) @ values.double().mul(scales.repeat_interleave(128, 1)).T)
