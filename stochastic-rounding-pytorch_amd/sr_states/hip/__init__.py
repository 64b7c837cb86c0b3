"""Fused gfx950 (MI355X) kernels: the HIP counterpart of ``sr_states.triton``."""

from ._common import is_hip_available
from .adamw import AdamWHip, AdamWHipRN, hip_adamw_step_
from .block import BlockScaled, block_cast, block_linear, block_matmul
from .cast import cast, rn_cast_bf16, sr_cast_bf16
from .muon import MuonHip, MuonHipRN, hip_muon_step_, orthogonalize
from .sgd import SGDMHip, SGDMHipRN, hip_sgdm_step_

__all__ = [
    "AdamWHip",
    "AdamWHipRN",
    "BlockScaled",
    "MuonHip",
    "MuonHipRN",
    "SGDMHip",
    "SGDMHipRN",
    "block_cast",
    "block_linear",
    "block_matmul",
    "cast",
    "hip_adamw_step_",
    "hip_muon_step_",
    "hip_sgdm_step_",
    "is_hip_available",
    "orthogonalize",
    "rn_cast_bf16",
    "sr_cast_bf16",
]
