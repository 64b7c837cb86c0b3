"""What the block casts' accesses promise about alignment, read from the IR of their own kernels (CPU).

Input rows start on any element and output rows on any byte, so an access may
promise one element's alignment at most; a GPU that takes any alignment shows
nothing at run time where one promises more.
"""

from __future__ import annotations

import os
import re
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
SIZES = {"ENC_F32": 4, "ENC_BF16_RN": 2, "ENC_F16_RN": 2}


@pytest.mark.parametrize("encoding", sorted(SIZES))
@pytest.mark.parametrize("kernel", ["block_cast_parts_kernel<sr::{}, sr::ENC_E4M3_RN>",
                                    "block_cast_tile_kernel<sr::{}, sr::ENC_E5M2_SR, false>",
                                    "block_cast_tile_kernel<sr::{}, sr::ENC_E4M3_RN, true>"])
def test_no_access_promises_more_than_an_element(tmp_path, kernel, encoding):
    source, listing = tmp_path / "cast.hip", tmp_path / "cast.ll"
    source.write_text('#include "sr_block_scaled.h"\n'
                      f"template __global__ void sr::{kernel.format(encoding)}(sr::BlockCastArgs);\n")
    subprocess.run([HIPCC, "--offload-arch=gfx950", "--cuda-device-only", "-O1", "-std=c++17", "-Xclang",
                    "-target-feature", "-Xclang", "-packed-fp32-ops", "-S", "-emit-llvm",
                    "-I", str(ROOT / "stochastic-rounding-pytorch_amd" / "csrc"), str(source), "-o", str(listing)],
                   check=True, stderr=subprocess.DEVNULL)
    text = listing.read_text()
    # The kernel's arguments are read in their own address space; these are the matrices.
    loads = re.findall(r"= load [^,\n]+, ptr addrspace\(1\) [^\n]*?align (\d+)", text)
    stores = re.findall(r"\bstore [^\n]*?, ptr addrspace\(1\) [^\n]*?align (\d+)", text)
    assert loads and max(map(int, loads)) <= SIZES[encoding]
    assert stores and max(map(int, stores)) == 1
