"""Shared launch plumbing: tensors -> raw pointers/strides -> C ABI call on the current stream."""

from __future__ import annotations

import array
import contextlib
import ctypes
from typing import ContextManager, Sequence

import torch

from .. import _hip


def ptr(t: torch.Tensor | None) -> ctypes.c_void_p:
    return ctypes.c_void_p(0 if t is None else t.data_ptr())


def require_gpu(t: torch.Tensor, who: str) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{who} runs on the GPU only; got a tensor on {t.device}")


# One cached scratch buffer per (device, stream): calls on one stream are serialised by the stream itself, so they can
# share scratch; different streams get different buffers.
_workspaces: dict[tuple[int, int], torch.Tensor] = {}


def workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    key = (device.index if device.index is not None else torch.cuda.current_device(),
           torch.cuda.current_stream(device).cuda_stream)
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = torch.empty(nbytes, device=device, dtype=torch.uint8)
        _workspaces[key] = ws
    return ws


def syrk_launch(
    mem_a: torch.Tensor,
    a_trans: bool,
    batch: int,
    n: int,
    k: int,
    c_mem: torch.Tensor | None,
    alpha: float,
    beta: float,
    d: torch.Tensor,
    skip_upper: bool,
) -> None:
    """``mem_a`` is the contiguous view of the operand: (B?, n, k) when not a_trans, else (B?, k, n)."""
    lib = _hip.lib()
    with torch.cuda.device(d.device):
        # scratch for the stream-K launch, when the library would use one for this shape
        nbytes = 0 if skip_upper else lib.mi_syrk_workspace_bytes(batch, n, k, int(a_trans))
        ws = workspace(d.device, nbytes) if nbytes else None
        rc = lib.mi_syrk_bf16_ws(
            ptr(mem_a), batch, n, k, n * k, mem_a.shape[-1], int(a_trans),
            ptr(c_mem), n * n, n, float(alpha), float(beta),
            ptr(d), n * n, n, int(bool(skip_upper)), ptr(ws), ws.numel() if ws is not None else 0,
            _hip.current_stream_ptr(d.device),
        )  # fmt: skip
    _hip.check(rc)


# ---------------------------------------------------------------------------------------------
# lists of tensors
# ---------------------------------------------------------------------------------------------
#: MI_DTYPE_* codes of the library
DTYPE_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def on_device(index: int) -> ContextManager:
    """Makes GPU ``index`` the current one, at no cost where it already is."""
    return contextlib.nullcontext() if torch.cuda.current_device() == index else torch.cuda.device(index)


def pointers(tensors: Sequence[torch.Tensor]) -> array.array:
    return array.array("q", map(torch.Tensor.data_ptr, tensors))


def address(a: array.array | None) -> int | None:
    return None if a is None else a.buffer_info()[0]


def is_dense(t: torch.Tensor) -> bool:
    """The elements fill one block of memory, in whatever order of the dimensions."""
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != want:
            return False
        want *= size
    return True


def list_device(who: str, *lists: Sequence[torch.Tensor]) -> int:
    """The one GPU all tensors of the lists are on."""
    found = set()
    for tensors in lists:
        found.update(map(torch.Tensor.get_device, tensors))
    if -1 in found:
        raise RuntimeError(f"{who} runs on the GPU only; got a tensor on the CPU")
    if len(found) != 1:
        raise ValueError(f"{who}: all tensors of a call must be on one GPU, got {sorted(found)}")
    return found.pop()


def list_dtype(who: str, what: str, tensors: Sequence[torch.Tensor], allowed: Sequence[torch.dtype] = tuple(DTYPE_CODES)) -> torch.dtype:
    """The one data type of the tensors of a list."""
    found = {t.dtype for t in tensors}
    if len(found) != 1 or not found <= set(allowed):
        names = ", ".join(sorted(str(d) for d in found))
        raise TypeError(f"{who}: {what} must have one data type out of {', '.join(str(d) for d in allowed)}, got {names}")
    return found.pop()


def check_like(who: str, what: str, tensors: Sequence[torch.Tensor], like: Sequence[torch.Tensor]) -> None:
    """``tensors`` have the shapes and the memory order of ``like``, whose elements fill their memory."""
    if len(tensors) != len(like):
        raise ValueError(f"{who}: {len(tensors)} {what} for {len(like)} params")
    for i, (t, p) in enumerate(zip(tensors, like)):
        if t.shape != p.shape:
            raise ValueError(f"{who}: {what}[{i}] has shape {tuple(t.shape)}, its param {tuple(p.shape)}")
        if not (t.is_contiguous() and p.is_contiguous()) and (t.stride() != p.stride() or not is_dense(p)):
            raise ValueError(f"{who}: {what}[{i}] must fill its memory in the order of its param, got strides {t.stride()} and {p.stride()}")
