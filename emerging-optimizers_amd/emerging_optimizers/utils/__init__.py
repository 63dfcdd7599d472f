"""Small helpers used on the orthogonalisation path."""

from __future__ import annotations

import contextlib
from typing import Iterable, Iterator, Literal, Union

import torch

from emerging_optimizers import hip_kernels
from emerging_optimizers.hip_kernels._launch import LIST_DTYPES, is_dense


__all__ = ["clip_grad_norm_", "fp32_matmul_precision", "FP32MatmulPrecT"]

FP32MatmulPrecT = Literal["highest", "high", "medium"]


@contextlib.contextmanager
def fp32_matmul_precision(precision: FP32MatmulPrecT = "highest") -> Iterator[None]:
    """Temporarily set ``torch.set_float32_matmul_precision`` (reference: utils/__init__.py:28-40).

    On this path the setting is more than a hint: ``"medium"`` is what switches ``newton_schulz`` to its
    bf16 kernels (muon_utils.py:245 of the reference).
    """
    saved = torch.get_float32_matmul_precision()
    torch.set_float32_matmul_precision(precision)
    try:
        yield
    finally:
        torch.set_float32_matmul_precision(saved)


@torch.no_grad()
def clip_grad_norm_(
    parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0, *, error_if_nonfinite: bool = False
) -> torch.Tensor:
    """Scales the gradients of ``parameters`` in place so that their global 2-norm is at most ``max_norm``.

    Same convention as ``torch.nn.utils.clip_grad_norm_`` (factor ``min(1, max_norm / (norm + 1e-6))``, the norm is
    returned as a float32 scalar; a gradient listed twice counts and is scaled twice) for its ``norm_type`` 2, the only one
    there is.  Gradients on one gfx950 GPU that fill their memory take two multi-tensor passes of the kernels
    (``hip_kernels.clip_grads_by_global_norm``) and nothing waits for the GPU unless ``error_if_nonfinite`` asks for
    the norm.
    """
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None]
    if norm_type != 2:
        raise ValueError(f"norm_type must be 2, got {norm_type}")
    if not max_norm >= 0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    if not grads:
        return torch.tensor(0.0)
    kernels = (
        hip_kernels.on_kernel_device(grads[0])
        and len(set(map(torch.Tensor.get_device, grads))) == 1
        and {g.dtype for g in grads}.issubset(LIST_DTYPES)
        and (all(map(torch.Tensor.is_contiguous, grads)) or all(map(is_dense, grads)))
    )
    if kernels and not error_if_nonfinite:
        try:
            return hip_kernels.clip_grads_by_global_norm(grads, max_norm=max_norm)
        except ValueError:  # memory that occurs twice, refused before anything is launched: the statements below take it
            kernels = False
    if kernels:
        norm, factor = hip_kernels.global_grad_norm(grads, max_norm=max_norm)
    else:
        norm = torch.stack([torch.linalg.vector_norm(g, dtype=torch.float64).to(grads[0].device) for g in grads]).square().sum().sqrt().float()
        factor = (max_norm / (norm + 1e-6)).clamp(max=1.0)
    if error_if_nonfinite and not bool(norm.isfinite()):
        raise RuntimeError(f"The global 2-norm of the gradients is {float(norm)}")
    if kernels:
        try:
            hip_kernels.scale_tensors(grads, factor)
            return norm
        except ValueError:  # as above
            pass
    for g in grads:
        g.mul_(factor.to(g.device))
    return norm
