"""Global 2-norm of a list of gradients, and scaling by it."""

from __future__ import annotations

from typing import Optional, Sequence, Union

import torch

from .. import _hip


__all__ = ["clip_grads_by_global_norm", "global_grad_norm", "scale_tensors"]


def global_grad_norm(grads: Sequence[torch.Tensor], *, max_norm: Optional[float] = None) -> Union[torch.Tensor, tuple[torch.Tensor, torch.Tensor]]:
    """2-norm over all elements of all ``grads`` (float32, bfloat16 and float16 may be mixed), as a float32 scalar on
    their GPU; sums in float64.  With ``max_norm`` also the factor ``min(1, max_norm / (norm + 1e-6))`` that clips to
    it, a float32 scalar on the GPU ready to be the ``grad_scale`` of :func:`fused_adamw_update`.  An infinite norm gives
    the factor 0, a norm that is not a number the factor NaN.  Nothing waits for the GPU.
    """
    if max_norm is not None and not max_norm >= 0:
        raise ValueError(f"global_grad_norm: max_norm must not be negative, got {max_norm}")
    rc, norm, factor = _hip.lists().global_norm("global_grad_norm", grads, 0.0 if max_norm is None else max_norm, False)
    _hip.check(rc)
    return norm if max_norm is None else (norm, factor)


def scale_tensors(tensors: Sequence[torch.Tensor], factor: torch.Tensor) -> None:
    """Multiplies every tensor in place by ``factor``, a float32 scalar on their GPU (nothing is touched if it is 1)."""
    _hip.check(_hip.lists().scale_tensors("scale_tensors", tensors, factor))


def clip_grads_by_global_norm(grads: Sequence[torch.Tensor], *, max_norm: float) -> torch.Tensor:
    """Scales all ``grads`` in place by ``min(1, max_norm / (norm + 1e-6))`` with ``norm`` their global 2-norm, which is
    returned (a float32 scalar on their GPU).  Nothing waits for the GPU; gradients within ``max_norm`` are not written.
    """
    if not max_norm >= 0:
        raise ValueError(f"clip_grads_by_global_norm: max_norm must not be negative, got {max_norm}")
    rc, norm, _ = _hip.lists().global_norm("clip_grads_by_global_norm", grads, max_norm, True)
    _hip.check(rc)
    return norm
