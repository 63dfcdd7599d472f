"""AdamW over lists of tensors: moments in 32 or in 8 bits, and the conversions of 8-bit moments."""

from __future__ import annotations

from typing import Literal, Optional, Sequence, Union

import torch

from .. import _hip


__all__ = ["fused_adamw_update", "fused_adamw_update_8bit", "moment_8bit_bytes", "pack_moments_8bit", "unpack_moments_8bit"]

MomentT = Literal["exp_avg", "exp_avg_sq"]
RoundingT = Literal["nearest", "dithered"]

_DECAY_METHODS = {"decoupled": 0, "independent": 1, "l2": 2, "palm": 3}
_MOMENTS = {"exp_avg": 0, "exp_avg_sq": 1}
_ROUNDING_BITS = {"nearest": 8, "dithered": 8 | 256}


def moment_8bit_bytes(numel: int) -> int:
    """Bytes of the 8-bit form of a moment of ``numel`` values: 64 codes and a float32 scale for each block of 64."""
    return -(-numel // 64) * 68


def _decay_code(method: str) -> int:
    code = _DECAY_METHODS.get(method)
    if code is None:
        raise ValueError(f"Invalid weight decay method: {method}")
    return code


def fused_adamw_update(
    params: Sequence[torch.Tensor],
    grads: Sequence[torch.Tensor],
    exp_avgs: Sequence[torch.Tensor],
    exp_avg_sqs: Sequence[torch.Tensor],
    *,
    step: Union[float, Sequence[torch.Tensor]],
    lr: Union[float, torch.Tensor],
    beta1: float,
    beta2: float,
    eps: float = 1e-8,
    weight_decay: float = 0.0,
    weight_decay_method: str = "decoupled",
    grad_scale: Optional[torch.Tensor] = None,
    model_params: Optional[Sequence[torch.Tensor]] = None,
) -> None:
    """One AdamW step of every tensor of ``params``, in place, with float32 moments (see ``mi_adamw_update``).

    ``g = grad_scale * grad`` (plus ``weight_decay * p`` for the method "l2"); ``m = beta1 * m + (1 - beta1) * g``;
    ``v = beta2 * v + (1 - beta2) * g**2``; ``p = keep * p - lr / (1 - beta1**t) * m / (sqrt(v / (1 - beta2**t)) + eps)``
    with ``keep`` by weight-decay method as in :class:`~emerging_optimizers.mixin.WeightDecayMixin`.  Everything is
    computed in float32 and rounded once.

    Args:
        params: weights of record; float32, bfloat16 or float16, one type a call, on one GPU
        grads: gradients; float32 or, where weights or ``model_params`` have 16 bits, that type; with float32 weights
            alone any of the three
        exp_avgs: first moments, float32
        exp_avg_sqs: second moments, float32
        step: number of this step, from 1; or one float32 tensor on the GPU for each param (captured graphs)
        lr: learning rate, a number or one float32 value on the GPU
        weight_decay_method: "decoupled", "independent", "l2" or "palm"
        grad_scale: one float32 value on the GPU that multiplies the gradients (``grads`` themselves stay as they are)
        model_params: 16-bit copies of float32 ``params``, written only

    Gradients, moments and copies have the shape of their param and fill their memory in its order; no tensor that is
    written may share memory with another one.  Any size from 0 on, any alignment.  The work is enqueued on the current
    stream of the tensors' GPU; nothing waits.
    """
    rc = _hip.lists().adamw_update(
        "fused_adamw_update", 32, params, grads, exp_avgs, exp_avg_sqs, model_params, step, lr, beta1, beta2, eps, weight_decay,
        _decay_code(weight_decay_method), grad_scale,
    )  # fmt: skip
    _hip.check(rc)


def fused_adamw_update_8bit(
    params: Sequence[torch.Tensor],
    grads: Sequence[torch.Tensor],
    exp_avgs: Sequence[torch.Tensor],
    exp_avg_sqs: Sequence[torch.Tensor],
    *,
    step: Union[float, Sequence[torch.Tensor]],
    lr: Union[float, torch.Tensor],
    beta1: float,
    beta2: float,
    eps: float = 1e-8,
    weight_decay: float = 0.0,
    weight_decay_method: str = "decoupled",
    grad_scale: Optional[torch.Tensor] = None,
    model_params: Optional[Sequence[torch.Tensor]] = None,
    rounding: RoundingT = "nearest",
) -> None:
    """:func:`fused_adamw_update` with moments in their 8-bit form: ``exp_avgs`` and ``exp_avg_sqs`` are uint8 tensors
    of :func:`moment_8bit_bytes` bytes each, 16-byte aligned (zeros stand for zero moments; see
    :func:`pack_moments_8bit`).  The update uses the new moments before they are rounded to 8 bits.

    ``rounding`` is how the new moments become codes.  "nearest" is the definition of :func:`pack_moments_8bit`, for single
    updates.  Over a run of steps it stops a moving average whose step is less than half the distance between two codes: with
    ``beta2=0.999`` a second moment whose gradients shrink never follows them while the largest one of its block stays.
    "dithered" is for training loops: from the fifth step on the code is the next one below or above, by an offset that rotates
    with ``step`` (see ``mi_adamw_update``), so moments follow on average (the root of a second one down to 1/1800 of its
    block's largest); consecutive calls need consecutive ``step``.
    """
    bits = _ROUNDING_BITS.get(rounding)
    if bits is None:
        raise ValueError(f'fused_adamw_update_8bit: rounding must be "nearest" or "dithered", got {rounding!r}')
    rc = _hip.lists().adamw_update(
        "fused_adamw_update_8bit", bits, params, grads, exp_avgs, exp_avg_sqs, model_params, step, lr, beta1, beta2, eps, weight_decay,
        _decay_code(weight_decay_method), grad_scale,
    )  # fmt: skip
    _hip.check(rc)


def _move(who: str, pack: bool, values: Sequence[torch.Tensor], packed: Sequence[torch.Tensor], which: MomentT) -> None:
    second = _MOMENTS.get(which)
    if second is None:
        raise ValueError(f'{who}: which must be "exp_avg" or "exp_avg_sq", got {which!r}')
    _hip.check(_hip.lists().move_moments(who, pack, values, packed, second))


def pack_moments_8bit(moments: Sequence[torch.Tensor], packed: Sequence[torch.Tensor], *, which: MomentT) -> None:
    """Writes the 8-bit form of every tensor of ``moments`` (float32, bfloat16 or float16) to its uint8 tensor of
    :func:`moment_8bit_bytes` bytes in ``packed``.

    The values, in memory order, are cut into blocks of 64 whose largest magnitude ``s`` is kept in float32.  ``which``
    is "exp_avg" (codes ``k`` from -127 to 127 for ``sign(k) * s * (k / 127)**2``) or "exp_avg_sq" (codes from 0 to 255
    for ``s * (k / 255)**4``, never 0 for a value over 0).  A block that holds a value that is not finite becomes NaN.
    """
    _move("pack_moments_8bit", True, moments, packed, which)


def unpack_moments_8bit(packed: Sequence[torch.Tensor], moments: Sequence[torch.Tensor], *, which: MomentT) -> None:
    """Writes the values that the 8-bit forms ``packed`` stand for to ``moments`` (float32, bfloat16 or float16)."""
    _move("unpack_moments_8bit", False, moments, packed, which)
