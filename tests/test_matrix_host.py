"""The matrix operators' C ABI surface and host-side checks (CPU)."""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest
import sr_states
import torch
from sr_states import _lib
from sr_states.hip.muon import _newton_schulz

HEADER = Path(__file__).resolve().parents[1] / "include" / "sr_matrix_hip.h"


def _declared():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    return sorted(set(re.findall(r"^\s*(?:int|int64_t)\s+(sr_\w+)\s*\(", text, flags=re.M)))


def test_library_exports_the_header():
    assert set(_declared()) == set(_lib.MATRIX_SIGNATURES)
    handle = _lib.library()
    for name in _declared():
        assert hasattr(handle, name), name
    assert handle.sr_matrix_abi_version() == _lib.MATRIX_ABI_VERSION
    text = HEADER.read_text()
    assert f"#define SR_MATRIX_ABI_VERSION {_lib.MATRIX_ABI_VERSION}" in text
    assert f"#define SR_BLOCK {_lib.BLOCK}" in text
    assert f"#define SR_MATRIX_BATCH {_lib.MATRIX_BATCH}" in text


def test_header_is_plain_c(tmp_path):
    import subprocess

    source = tmp_path / "sizes.c"
    source.write_text(
        f'#include "{HEADER}"\n#include <stdio.h>\n'
        "int main(void) { printf(\"%zu %zu %zu %zu %zu\", sizeof(sr_block_matrix), sizeof(sr_block_output),"
        " sizeof(sr_newton_schulz), sizeof(sr_muon_row), sizeof(sr_muon_hparams)); return 0; }\n"
    )
    program = tmp_path / "sizes"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", str(source), "-o", str(program)], check=True)
    sizes = [int(n) for n in subprocess.run([str(program)], capture_output=True, text=True, check=True).stdout.split()]
    assert sizes == [ctypes.sizeof(s) for s in (_lib.BlockMatrix, _lib.BlockOutput, _lib.NewtonSchulz, _lib.MuonRow,
                                                _lib.MuonHparams)]


def _matrix(**changes):
    fields = {"data": 1 << 20, "scale": 1 << 20, "ld": 128, "ld_scale": 1, "rows": 4, "dtype": _lib.SR_E4M3,
              "scale_type": 0, "block_rows": 1, **changes}
    return _lib.BlockMatrix(**fields)


def test_invalid_arguments_fail_before_any_device_work():
    lib = _lib.library()
    good = _matrix()

    def matmul(a=good, b=good, k=128, out=1 << 20, ldo=4, dtype=_lib.SR_BF16):
        return lib.sr_block_matmul(a, b, k, out, ldo, dtype, None)

    for call, message in [
        (lambda: matmul(a=_matrix(dtype=_lib.SR_BF16)), b"E4M3 or E5M2"),
        (lambda: matmul(a=_matrix(scale_type=2)), b"scale type"),
        (lambda: matmul(b=_matrix(block_rows=64)), b"1 or 128 rows"),
        (lambda: matmul(b=_matrix(rows=-1)), b"-1 rows"),
        (lambda: matmul(b=_matrix(ld=100)), b"bytes between rows"),
        (lambda: matmul(b=_matrix(ld=1 << 25)), b"bytes between rows"),
        (lambda: matmul(b=_matrix(ld_scale=1 << 21)), b"scales between rows"),
        (lambda: matmul(b=_matrix(data=None)), b"null pointer"),
        (lambda: matmul(b=_matrix(scale_type=1)), b"different scale types"),
        (lambda: matmul(a=None), b"null argument"),
        (lambda: matmul(k=-1), b"contracted"),
        (lambda: matmul(dtype=_lib.SR_E4M3), b"FP32, BF16 or FP16"),
        (lambda: matmul(out=None), b"null pointer"),
        (lambda: matmul(ldo=3), b"overlap"),
    ]:
        assert call() == 1
        assert message in lib.sr_last_error()
    assert matmul(a=_matrix(rows=0, data=None, scale=None)) == 0  # empty: nothing to do

    out = _lib.BlockOutput(1 << 20, 1 << 20, 256, 2)

    def cast(x=1 << 20, ldx=256, rows=4, cols=256, x_dtype=0, dtype=_lib.SR_E4M3, rule=1, by_rows=out, by_cols=None):
        return lib.sr_block_cast(x, ldx, rows, cols, x_dtype, dtype, rule, 0, 0, 0, by_rows, by_cols, None)

    for call, message in [
        (lambda: cast(x_dtype=_lib.SR_E4M3), b"FP32, BF16 or FP16"),
        (lambda: cast(dtype=_lib.SR_F16), b"E4M3 or E5M2"),
        (lambda: cast(rule=2), b"rounding rule"),
        (lambda: cast(rows=-1), b"matrix"),
        (lambda: cast(by_rows=None), b"no output"),
        (lambda: cast(x=None), b"null pointer"),
        (lambda: cast(ldx=255), b"overlap"),
        (lambda: cast(by_cols=_lib.BlockOutput(1 << 20, 1 << 20, 3, 1)), b"overlap"),
        (lambda: cast(by_cols=_lib.BlockOutput(1 << 20, None, 4, 1)), b"null pointer"),
    ]:
        assert call() == 1
        assert message in lib.sr_last_error()
    assert cast(rows=0) == 0

    ns = _newton_schulz(5, (3.4445, -4.7750, 2.0315), 1e-7)
    bad = _lib.NewtonSchulz(1.0, 0.0, 0.0, 0.0, 0)
    hp = _lib.MuonHparams(0.9, 1.0, -0.1, 1)
    rows = (_lib.MuonRow * 1)(_lib.MuonRow(1 << 20, 1 << 20, None, 0, 0))
    for call, message in [
        (lambda: lib.sr_orthogonalize(1, 1, 1, 0, 0, 4, 4, 0, 0, bad, 1, None), b"steps"),
        (lambda: lib.sr_orthogonalize(1, 1, -1, 0, 0, 4, 4, 0, 0, ns, 1, None), b"negative"),
        (lambda: lib.sr_orthogonalize(1, 1, 1, 0, 0, 1 << 21, 4, 0, 0, ns, 1, None), b"too large"),
        (lambda: lib.sr_orthogonalize(1, 1, 1, 0, 0, 4, 4, 3, 0, ns, 1, None), b"FP32, BF16 or FP16"),
        (lambda: lib.sr_orthogonalize(1, 1, 1, 0, 0, 4, 4, 0, 0, ns, None, None), b"null pointer"),
        (lambda: lib.sr_orthogonalize(1, 1, 2, 16, 15, 4, 4, 0, 0, ns, 1, None), b"overlap"),
        (lambda: lib.sr_muon_multi(rows, 1, 4, 4, 2, 0, 1, 1, hp, ns, 1, None), b"FP32 or BF16"),
        (lambda: lib.sr_muon_multi(rows, 1, 4, 4, 0, 0, 9, 1, hp, ns, 1, None), b"unsupported state"),
        (lambda: lib.sr_muon_multi(rows, 1, 4, 4, 0, 0, 1, 1, None, ns, 1, None), b"null hyperparameters"),
        (lambda: lib.sr_muon_multi(rows, 1, 4, 4, 0, 0, 1, 1, hp, ns, 1, None), b"row 0: null pointer"),
    ]:
        assert call() == 1
        assert message in lib.sr_last_error()
    assert lib.sr_orthogonalize(None, None, 0, 0, 0, 4, 4, 0, 0, ns, None, None) == 0


def test_operators_refuse_cpu_tensors():
    x = torch.zeros(4, 256)
    q = sr_states.BlockScaled(x.to(torch.float8_e4m3fn), torch.ones(4, 2))
    for call in (lambda: sr_states.block_cast(x), lambda: sr_states.orthogonalize(x),
                 lambda: sr_states.block_matmul(q, q), lambda: sr_states.block_linear(x, x),
                 lambda: sr_states.hip_muon_step_(x, x.clone(), x.clone(), lr=0.1, momentum_factor=0.9, seed=0)):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_public_names():
    for name in ("BlockScaled", "block_cast", "block_matmul", "block_linear", "orthogonalize", "hip_muon_step_",
                 "MuonHip", "MuonHipRN"):
        assert name in sr_states.__all__ and name in sr_states.hip.__all__


def test_dequantize():
    data = torch.ones(130, 200).to(torch.float8_e5m2)
    rows = sr_states.BlockScaled(data, torch.arange(260.0).view(130, 2)).dequantize()
    assert rows.shape == (130, 200) and rows[3, 127] == 6 and rows[3, 128] == 7
    square = sr_states.BlockScaled(data, torch.tensor([[1.0, 2.0], [3.0, 4.0]])).dequantize()
    assert square[127, 0] == 1 and square[128, 0] == 3 and square[129, 199] == 4


def test_coefficients_are_checked_over_every_singular_value():
    _newton_schulz(5, (3.4445, -4.7750, 2.0315), 1e-7)
    _newton_schulz(30, (1.5, -0.5, 0.0), 0.0)
    for bad in ((3.0, 0.0, 0.0), (1.0, 8.0, 0.0), (5.0, -9.0, 4.0), (float("nan"), 0.0, 0.0)):
        with pytest.raises(ValueError):
            _newton_schulz(5, bad, 1e-7)
    with pytest.raises(ValueError):
        _newton_schulz(True, (1.5, -0.5, 0.0), 0.0)


def test_workspace_grows_with_the_batch_up_to_a_launch():
    size = _lib.library().sr_orthogonalize_workspace
    one = size(1, 100, 200)
    # Ten bytes per padded element, four per padded Gram entry, and partial sums.
    assert one == 128 * 256 * 10 + 128 * 128 * 4 + 2048
    assert size(3, 200, 100) > 2 * one
    assert size(64, 100, 200) == size(65, 100, 200) == size(1000, 100, 200)
    assert size(0, 100, 200) == size(1, 0, 5) == 0


@pytest.mark.parametrize("options, message", [
    ({"lr": -1.0}, "learning rate"),
    ({"momentum": 1.0}, "momentum"),
    ({"weight_decay": float("nan")}, "weight_decay"),
    ({"update_scale": "adam"}, "update_scale"),
    ({"ns_steps": 0}, "steps"),
    ({"ns_coefficients": (9.0, 0.0, 0.0)}, "out of range"),
])
def test_optimizer_rejects_invalid_options(options, message):
    with pytest.raises(ValueError, match=message):
        sr_states.MuonHip([torch.nn.Parameter(torch.zeros(4, 4))], **options)


def test_optimizer_takes_matrices_only():
    vector = torch.nn.Parameter(torch.zeros(4))
    with pytest.raises(ValueError, match="one dimension"):
        sr_states.MuonHip([vector])
    opt = sr_states.MuonHip([{"params": (torch.nn.Parameter(torch.zeros(4, 4)) for _ in range(2))}])
    assert len(opt.param_groups[0]["params"]) == 2
    with pytest.raises(ValueError, match="one dimension"):
        opt.add_param_group({"params": vector})
    opt.add_param_group({"params": torch.nn.Parameter(torch.zeros(2, 3, 1, 1)), "lr": 0.5})
    assert opt.param_groups[1]["lr"] == 0.5 and opt.param_groups[1]["momentum"] == 0.95


def test_optimizer_checkpoints_before_the_first_step():
    parameter = torch.nn.Parameter(torch.zeros(4, 4))
    opt = sr_states.MuonHip([parameter], lr=0.1, state_dtype=torch.float8_e5m2, seed=5)
    other = sr_states.MuonHip([torch.nn.Parameter(torch.zeros(4, 4))])
    other.load_state_dict(opt.state_dict())
    group = other.param_groups[0]
    assert group["lr"] == 0.1 and group["sr_seed"] == 5
    assert group["state_format"]["momentum_buffer"]["dtype"] == torch.float8_e5m2
    assert sr_states.MuonHipRN([parameter]).param_groups[0]["state_format"]["momentum_buffer"]["rounding"] == "nearest"
