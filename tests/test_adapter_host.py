"""The adapters' C ABI checks, refusals without a GPU, and their oracle (CPU)."""

from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import _adapter_oracle as oracle
import pytest
import sr_states
import torch
from sr_states import _lib

HEADER = Path(__file__).resolve().parents[1] / "include" / "sr_matrix_hip.h"


def test_structures_and_constants_match_the_header(tmp_path):
    source = tmp_path / "sizes.c"
    source.write_text(
        f'#include "{HEADER}"\n#include <stdio.h>\n'
        'int main(void) { printf("%zu %d", sizeof(sr_adapters), SR_MATRIX_ADAPTERS); return 0; }\n'
    )
    program = tmp_path / "sizes"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", str(source), "-o", str(program)], check=True)
    sizes = [int(n) for n in subprocess.run([str(program)], capture_output=True, text=True, check=True).stdout.split()]
    assert sizes == [ctypes.sizeof(_lib.AdapterSet), _lib.MATRIX_ADAPTERS]


def _adapters(**changes):
    fields = {"a": 1 << 20, "b": 1 << 20, "index": 1 << 20, "scaling": None, "scale": 1.0, "count": 2, "rank": 8,
              "dtype": _lib.SR_BF16, "wide": 0, **changes}
    return _lib.AdapterSet(**fields)


def test_invalid_arguments_fail_before_any_device_work():
    lib = _lib.library()
    good, p = _adapters(), 1 << 20

    def add(g=good, x=p, ldx=64, k=64, base=p, ldbase=32, n=32, rows=4, out=p, ldo=32, low=p):
        return lib.sr_adapter_add(g, x, ldx, k, base, ldbase, n, rows, out, ldo, low, None)

    def backward(g=good, x=p, ldx=64, dy=p, lddy=32, low=p, dx=p, lddx=64, da=p, db=p, workspace=p, rows=4):
        return lib.sr_adapter_backward(g, x, ldx, 64, dy, lddy, 32, rows, low, dx, lddx, da, db, workspace, None)

    for call, message in [
        (lambda: add(g=None), b"null argument"),
        (lambda: add(g=_adapters(dtype=_lib.SR_E4M3)), b"FP32, BF16 or FP16"),
        (lambda: add(g=_adapters(rank=0)), b"rank 0"),
        (lambda: add(g=_adapters(rank=129)), b"rank 129"),
        (lambda: add(g=_adapters(count=-1)), b"-1 adapters"),
        (lambda: add(g=_adapters(count=65537)), b"65537 adapters"),
        (lambda: add(g=_adapters(a=None)), b"null pointer"),
        (lambda: add(g=_adapters(b=None)), b"null pointer"),
        (lambda: add(g=_adapters(index=None)), b"null pointer"),
        (lambda: add(rows=-1), b"-1 rows"),
        (lambda: add(k=(1 << 24) + 1), b"rows"),
        (lambda: add(ldx=63), b"overlap"),
        (lambda: add(ldbase=31), b"overlap"),
        (lambda: add(ldo=31), b"overlap"),
        (lambda: add(x=None), b"null pointer"),
        (lambda: add(base=None), b"null pointer"),
        (lambda: add(out=None), b"null pointer"),
        (lambda: add(low=None), b"null pointer"),
        (lambda: backward(g=_adapters(rank=129)), b"rank 129"),
        (lambda: backward(ldx=63), b"overlap"),
        (lambda: backward(lddy=31), b"overlap"),
        (lambda: backward(lddx=63), b"overlap"),
        (lambda: backward(x=None), b"null pointer"),
        (lambda: backward(dy=None), b"null pointer"),
        (lambda: backward(low=None), b"null pointer"),
        (lambda: backward(workspace=None), b"null pointer"),
    ]:
        assert call() == 1
        assert message in lib.sr_last_error()
    assert add(rows=0, x=None) == 0  # empty: nothing to do
    assert backward(dx=None, da=None, db=None) == 0


def test_workspaces_cover_the_shapes_that_are_taken():
    low, workspace = _lib.library().sr_adapter_low, _lib.library().sr_adapter_workspace
    assert low(8192, 2048, 16, _lib.SR_BF16) == 8192 * 16  # rows enough for every CU
    assert low(1, 2048, 8, _lib.SR_BF16) == 4 * 16  # four parts of one row, eight waves and a step each
    assert low(1, 1, 17, _lib.SR_F32) == 32
    assert low(4, 64, 129, _lib.SR_F32) == low(-1, 64, 8, _lib.SR_F32) == low(4, 64, 8, _lib.SR_E4M3) == 0
    turned = 4 * 8 * (2048 + 512) * 2
    assert workspace(100, 2048, 512, 4, 8, _lib.SR_BF16) >= turned + 4 * low(100, 512, 8, _lib.SR_BF16)
    assert workspace(100000, 2048, 512, 4, 8, _lib.SR_BF16) < turned + 4 * 100000 * 16 + (257 << 20)
    assert workspace(100, 2048, 512, 4, 0, _lib.SR_BF16) == 0


def test_operators_refuse_cpu_tensors():
    x, a, b, index = torch.zeros(4, 20), torch.zeros(2, 3, 20), torch.zeros(2, 5, 3), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        sr_states.adapter_add(torch.zeros(4, 5), x, a, b, index)


def test_public_names():
    assert "adapter_add" in sr_states.__all__ and "adapter_add" in sr_states.hip.__all__


def test_the_oracle_is_the_gradient_of_its_result():
    gen = torch.Generator().manual_seed(2)
    base, x, a, b = (torch.randn(s, generator=gen, dtype=torch.float64) for s in ((7, 6), (7, 5), (3, 2, 5), (3, 6, 2)))
    index, scaling, dy = torch.tensor([0, 2, -1, 2, 0, 5, 1]), torch.tensor([0.5, -2.0, 1.5]), torch.randn(7, 6, generator=gen, dtype=torch.float64)
    for t in (x, a, b):
        t.requires_grad_()
    y = base.clone()
    rows = [y[t] if not 0 <= i < 3 else y[t] + scaling[i].double() * (b[i] @ (a[i] @ x[t])) for t, i in enumerate(index.tolist())]
    y = torch.stack(rows)
    value, size = oracle.add(base, x, a, b, index, scaling)
    torch.testing.assert_close(value, y.detach())
    assert (size >= value.abs() - 1e-12).all()
    for (got, size), want in zip(oracle.gradients(dy, x, a, b, index, scaling), torch.autograd.grad(y, (x, a, b), dy)):
        torch.testing.assert_close(got, want)
        assert (size >= got.abs() - 1e-12).all()
