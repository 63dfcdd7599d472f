"""Global 2-norm of a list of gradients, and scaling by it."""

from __future__ import annotations

from typing import Optional, Sequence, Union

import torch

from .. import _hip
from . import _launch


__all__ = ["clip_grads_by_global_norm", "global_grad_norm", "scale_tensors"]


class _List:
    """Host arrays of a checked list of dense tensors on one GPU."""

    def __init__(self, who: str, tensors: Sequence[torch.Tensor]) -> None:
        try:
            codes = [_launch.DTYPE_CODES[t.dtype] for t in tensors]
        except KeyError as exc:
            raise TypeError(f"{who}: tensors must be float32, bfloat16 or float16, got {exc.args[0]}") from None
        if not all(map(torch.Tensor.is_contiguous, tensors)) and not all(map(_launch.is_dense, tensors)):
            raise ValueError(f"{who}: tensors must fill their memory")
        self.device = _launch.list_device(who, tensors)
        self.arrays = [
            _launch.pointers(tensors),
            _launch.array.array("q", map(torch.Tensor.numel, tensors)),
            _launch.array.array("i", codes),
        ]
        self.count = len(tensors)

    def args(self) -> list:
        return [self.count, *map(_launch.address, self.arrays)]


def _norm(t: _List, max_norm: float) -> torch.Tensor:
    """(norm, factor) as one tensor of two values."""
    lib = _hip.lib()
    length = lib.mi_global_norm_partials_len(t.count, _launch.address(t.arrays[1]))
    out = torch.empty(2, device=t.device, dtype=torch.float32)
    # Scratch of this call alone: taken from the caching allocator for the current stream (and from a graph's own pool
    # while one is captured), so no two calls or graphs share it.
    partials = torch.empty(length, device=t.device, dtype=torch.float64)
    rc = lib.mi_global_norm(
        *t.args(), float(max_norm), partials.data_ptr() if length else None, length, out.data_ptr(), torch.cuda.current_stream().cuda_stream
    )
    _hip.check(rc)
    return out


def global_grad_norm(grads: Sequence[torch.Tensor], *, max_norm: Optional[float] = None) -> Union[torch.Tensor, tuple[torch.Tensor, torch.Tensor]]:
    """2-norm over all elements of all ``grads`` (float32, bfloat16 and float16 may be mixed), as a float32 scalar on
    their GPU; sums in float64.  With ``max_norm`` also the factor ``min(1, max_norm / (norm + 1e-6))`` that clips to
    it, a float32 scalar on the GPU ready to be the ``grad_scale`` of :func:`fused_adamw_update`.  An infinite norm gives
    the factor 0, a norm that is not a number the factor NaN.  Nothing waits for the GPU.
    """
    if max_norm is not None and not max_norm >= 0:
        raise ValueError(f"global_grad_norm: max_norm must not be negative, got {max_norm}")
    if len(grads) == 0:
        raise ValueError("global_grad_norm needs at least one tensor")
    t = _List("global_grad_norm", grads)
    with _launch.on_device(t.device):
        norm, factor = _norm(t, 0.0 if max_norm is None else max_norm).unbind()
    return norm if max_norm is None else (norm, factor)


def scale_tensors(tensors: Sequence[torch.Tensor], factor: torch.Tensor) -> None:
    """Multiplies every tensor in place by ``factor``, a float32 scalar on their GPU (nothing is touched if it is 1)."""
    if len(tensors) == 0:
        return
    t = _List("scale_tensors", tensors)
    if factor.dtype != torch.float32 or factor.numel() != 1 or factor.get_device() != t.device:
        raise ValueError(f"scale_tensors: factor must be one float32 value on the GPU of the tensors, got {factor.dtype} {tuple(factor.shape)} on {factor.device}")
    with _launch.on_device(t.device):
        _hip.check(_hip.lib().mi_scale_tensors(*t.args(), factor.data_ptr(), torch.cuda.current_stream().cuda_stream))


def clip_grads_by_global_norm(grads: Sequence[torch.Tensor], *, max_norm: float) -> torch.Tensor:
    """Scales all ``grads`` in place by ``min(1, max_norm / (norm + 1e-6))`` with ``norm`` their global 2-norm, which is
    returned (a float32 scalar on their GPU).  Nothing waits for the GPU; gradients within ``max_norm`` are not written.
    """
    if not max_norm >= 0:
        raise ValueError(f"clip_grads_by_global_norm: max_norm must not be negative, got {max_norm}")
    if len(grads) == 0:
        raise ValueError("clip_grads_by_global_norm needs at least one tensor")
    t = _List("clip_grads_by_global_norm", grads)
    with _launch.on_device(t.device):
        out = _norm(t, max_norm)
        _hip.check(_hip.lib().mi_scale_tensors(*t.args(), out.data_ptr() + 4, torch.cuda.current_stream().cuda_stream))
    return out[0]
