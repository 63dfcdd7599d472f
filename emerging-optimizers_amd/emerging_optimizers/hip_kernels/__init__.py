"""Python entry points of the gfx950 kernels (SYRK, GEMM+AXPY, Frobenius normalise, fused Newton-Schulz, AdamW over
lists of tensors)."""

from .. import _hip
from .adamw import (
    fused_adamw_update,
    fused_adamw_update_8bit,
    moment_8bit_bytes,
    pack_moments_8bit,
    unpack_moments_8bit,
)
from .batched_syrk import batched_tsyrk_ex, can_use_batched_tsyrk
from .grad_norm import clip_grads_by_global_norm, global_grad_norm, scale_tensors
from .newton_schulz import (
    frob_normalize,
    fused_muon_update,
    fused_newton_schulz,
    fused_supported,
    gemm_axpy,
    on_kernel_device,
    require_library,
)
from .syrk import tsyrk_ex, tsyrk_ex_small_matrix


#: True when libmi_ns.so is loadable.  The reference's call sites test ``HAS_TRITON_340`` before taking
#: the SYRK path (muon.py:106, muon_utils.py:431,465); the same attribute name is kept for them.
HAS_HIP_KERNELS = _hip.available()
HAS_TRITON_340 = HAS_HIP_KERNELS

__all__ = [
    "HAS_HIP_KERNELS",
    "HAS_TRITON_340",
    "batched_tsyrk_ex",
    "can_use_batched_tsyrk",
    "clip_grads_by_global_norm",
    "frob_normalize",
    "fused_adamw_update",
    "fused_adamw_update_8bit",
    "fused_muon_update",
    "fused_newton_schulz",
    "fused_supported",
    "gemm_axpy",
    "global_grad_norm",
    "moment_8bit_bytes",
    "on_kernel_device",
    "pack_moments_8bit",
    "require_library",
    "scale_tensors",
    "tsyrk_ex",
    "tsyrk_ex_small_matrix",
    "unpack_moments_8bit",
]
