"""B200-native (sm_100a) implementation of the MoE-layer hot path of open-lm-engine/cute-kernels.

Drop-in names: `MoE`, `Experts`, `continuous_count`, `grouped_gemm`, `swiglu`, `swiglu_packed`,
`pack_sequence`, `unpack_sequence`, `KernelBackend`.  All compute runs in hand-written CUDA kernels loaded from libfma_b200.so through a
C ABI (see include/fma_b200.h); there is no Triton, eager-PyTorch or CPU fallback.
"""

from . import _native
from .kernel_backend import KernelBackend
from .modules import Experts, ExpertParallelMoE, MoE, shard_expert_state_dict, unshard_expert_state_dicts
from .ops import (
    continuous_count,
    grouped_gemm,
    grouped_linear_fp8,
    linear_fp8,
    pack_sequence,
    quantize_fp8,
    quantize_fp8_weight,
    swiglu,
    swiglu_fp8_checkpoint,
    swiglu_packed,
    unpack_sequence,
)
from .utils import ceil_divide, ensure_contiguous, set_seed

__all__ = [
    "KernelBackend",
    "MoE",
    "Experts",
    "ExpertParallelMoE",
    "shard_expert_state_dict",
    "unshard_expert_state_dicts",
    "continuous_count",
    "grouped_gemm",
    "swiglu",
    "swiglu_packed",
    "pack_sequence",
    "unpack_sequence",
    "quantize_fp8",
    "quantize_fp8_weight",
    "linear_fp8",
    "grouped_linear_fp8",
    "swiglu_fp8_checkpoint",
    "ensure_contiguous",
    "set_seed",
    "ceil_divide",
]


def __getattr__(name: str):
    if name in ("Fp8Blocks", "Fp8Weight"):  # what quantize_fp8 and quantize_fp8_weight return
        return getattr(_native.binding(), name)
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
