"""Fused gfx950 (MI355X) kernels: the HIP counterpart of ``sr_states.triton``."""

from ._common import is_hip_available
from .adamw import AdamWHip, AdamWHipRN, hip_adamw_step_
from .adapter import adapter_add
from .block import BlockScaled, block_cast, block_linear, block_matmul
from .cast import cast, rn_cast_bf16, sr_cast_bf16
from .grouped import grouped_block_cast, grouped_block_linear, grouped_block_matmul
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
    "adapter_add",
    "block_cast",
    "block_linear",
    "block_matmul",
    "cast",
    "grouped_block_cast",
    "grouped_block_linear",
    "grouped_block_matmul",
    "hip_adamw_step_",
    "hip_muon_step_",
    "hip_sgdm_step_",
    "is_hip_available",
    "orthogonalize",
    "rn_cast_bf16",
    "sr_cast_bf16",
]
