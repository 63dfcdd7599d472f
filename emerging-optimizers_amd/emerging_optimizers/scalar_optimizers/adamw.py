"""AdamW for the parameters that are not orthogonalised: embeddings, the output head, gains and biases.

All parameters of one kind are updated by one multi-tensor call (``hip_kernels.fused_adamw_update`` or, with
``moment_bits=8``, ``hip_kernels.fused_adamw_update_8bit``).  The reference leaves these parameters to
``torch.optim.AdamW``; the defaults and the names of the state's entries are those of that class, so checkpoints move
in both directions.  Weight decay has the methods of the other optimizers of this package.

On the CPU, on GPUs other than gfx950, for float64 parameters and for a bfloat16 parameter with a float16 gradient (or the
other way round) the same formulas run as torch statements.
"""

from __future__ import annotations

from typing import Any, Callable, Optional, Union

import torch
from torch.optim.optimizer import Optimizer, ParamsT

from emerging_optimizers import hip_kernels
from emerging_optimizers.hip_kernels._launch import LIST_DTYPES, is_dense
from emerging_optimizers.mixin import WeightDecayMixin, WeightDecayT


__all__ = ["AdamW"]

_BLOCK = 64  # values that share a scale in the 8-bit form of a moment
_SMALLEST = torch.finfo(torch.float32).tiny
# how far the offset of a dithered code rotates with the step and from place to place, in 2^-32 turns
_ROTATION = {"exp_avg": (0x9E3779B9, 0x6A09E667), "exp_avg_sq": (0x6A09E667, 0xBB67AE85)}


def _offsets(numel: int, which: str, step: Union[int, torch.Tensor], device: torch.device) -> torch.Tensor:
    """Offset in [0, 1) that each of ``numel`` places adds before its code is rounded down; 1/2, to nearest, in the
    first four steps."""
    by_step, by_place = _ROTATION[which]
    turns = torch.arange(numel, device=device) * by_place
    if isinstance(step, torch.Tensor):
        turns = torch.where(step > 4, turns + step.long() * by_step, 1 << 31)
    else:
        turns = turns + step * by_step if step > 4 else torch.full_like(turns, 1 << 31)
    return ((turns & 0xFFFFFFFF) >> 9).float() * 2.0**-23


def _pack_torch(x: torch.Tensor, which: str, step: Union[None, int, torch.Tensor] = None) -> torch.Tensor:
    """``hip_kernels.pack_moments_8bit`` as torch statements: the 8-bit form of the flat float32 ``x``; with ``step`` the
    dithered codes of that step of ``hip_kernels.fused_adamw_update_8bit``."""
    blocks = torch.nn.functional.pad(x, (0, -x.numel() % _BLOCK)).view(-1, _BLOCK)
    scale = blocks.abs().amax(1, keepdim=True)
    scale = torch.where(scale.isfinite(), torch.where(scale < _SMALLEST, 0.0, scale), torch.nan)
    share = torch.where(scale > 0, blocks.abs() / scale, 0.0)
    first = which == "exp_avg"
    codes = share.sqrt() * 127 if first else share.sqrt().sqrt() * 255
    if step is None:
        codes = codes.round()
    else:
        up = _offsets(blocks.numel(), which, step, x.device).view_as(blocks)
        if not first:  # below code 6 upwards: a root of v held at a fraction of itself would blow the update up
            up = torch.where((codes < 6) & (torch.as_tensor(step, device=x.device) > 4), 255 / 256, up)
        codes = (codes + up).floor().clamp_max(127 if first else 255)
    if first:
        codes = (codes * blocks.sign()).nan_to_num().to(torch.int8).view(torch.uint8)
    else:
        codes = torch.where((scale > 0) & (blocks > 0), codes.clamp_min(1), codes).nan_to_num().to(torch.uint8)
    return torch.cat([codes.view(-1), scale.view(-1).view(torch.uint8)])


def _unpack_torch(packed: torch.Tensor, numel: int, which: str) -> torch.Tensor:
    """``hip_kernels.unpack_moments_8bit`` as torch statements: flat float32 values."""
    size = packed.numel() // (_BLOCK + 4) * _BLOCK
    codes, scale = packed[:size], packed[size:].clone().view(torch.float32).repeat_interleave(_BLOCK)
    if which == "exp_avg":
        k = codes.view(torch.int8).float()
        return (k * k.abs() * (1 / 127**2) * scale)[:numel]
    k = codes.float().square() * (1 / 255**2)
    return (k * k * scale)[:numel]


class AdamW(WeightDecayMixin, Optimizer):
    """Adam with decoupled weight decay (arXiv:1711.05101), one call for all parameters of a kind.

    Args:
        params: parameters (or parameter-group dicts) to optimize; float32, bfloat16 or float16 on a gfx950 GPU run on
            the kernels
        lr: learning rate; a number or, with ``capturable``, also one float32 value on the GPU
        betas: EMA coefficients of gradient and squared gradient
        eps: added to the square root of the second moment
        weight_decay: weight-decay strength; how it is applied is set by ``weight_decay_method``
        weight_decay_method: one of the flavours of :class:`~emerging_optimizers.mixin.WeightDecayMixin`
        moment_bits: 32 for float32 moments, 8 for one byte a value and a float32 scale for each 64 values
            (``hip_kernels.pack_moments_8bit``), dithered so that moments follow the gradients on average
            (``rounding="dithered"`` of ``hip_kernels.fused_adamw_update_8bit``); 8 saves 5.9 bytes a parameter.  Updates
            differ from the 32-bit ones by a few per cent where the gradients of a block of 64 are of similar size (simulated
            2.5 to 6 % for scales spread as exp(N(0, 0.5))), by 12 to 16 % for exp(N(0, 1.5)) and by 40 % for exp(N(0, 2.5))
        master_weights: keep float32 weights of record for 16-bit parameters (in the state, as ``master``); without them
            a step smaller than half the distance between neighbouring 16-bit numbers is lost
        capturable: keep the step count on the GPU, so that a captured ``step()`` counts on when it is replayed
    """

    def __init__(
        self,
        params: ParamsT,
        lr: float = 1e-3,
        betas: tuple[float, float] = (0.9, 0.999),
        eps: float = 1e-8,
        weight_decay: float = 0.01,
        *,
        weight_decay_method: WeightDecayT = "decoupled",
        moment_bits: int = 32,
        master_weights: bool = False,
        capturable: bool = False,
    ) -> None:
        if moment_bits not in (8, 32):
            raise ValueError(f"moment_bits must be 8 or 32, got {moment_bits}")
        if weight_decay_method not in ("decoupled", "independent", "l2", "palm"):
            raise ValueError(f"Invalid weight decay method: {weight_decay_method}")
        self.weight_decay_method = weight_decay_method
        self.moment_bits = moment_bits
        self.master_weights = bool(master_weights)
        self.capturable = bool(capturable)
        defaults = dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay)
        self._check_options(defaults)
        super().__init__(params, defaults)

    def _check_options(self, options: dict) -> None:
        betas, lr = options["betas"], options["lr"]
        if not 0.0 <= betas[0] < 1.0 or not 0.0 <= betas[1] < 1.0:
            raise ValueError(f"betas must be in [0, 1), got {betas}")
        if not options["eps"] >= 0.0:
            raise ValueError(f"eps must not be negative, got {options['eps']}")
        if isinstance(lr, torch.Tensor) and not self.capturable:
            raise ValueError("a learning rate in a tensor needs capturable=True")
        if not lr >= 0.0:
            raise ValueError(f"the learning rate must not be negative, got {lr}")

    def add_param_group(self, param_group: dict) -> None:
        """Adds a group, whose own options are checked as the constructor's are."""
        if isinstance(param_group, dict):
            self._check_options({**self.defaults, **param_group})
        super().add_param_group(param_group)

    def __getstate__(self) -> dict:
        # the base class copies and pickles options, state and parameter groups only
        own = ("weight_decay_method", "moment_bits", "master_weights", "capturable")
        return {**super().__getstate__(), **{name: getattr(self, name) for name in own}}

    def _moment(self, p: torch.Tensor) -> torch.Tensor:
        """A zero moment of ``p``."""
        if self.moment_bits == 8:
            return torch.zeros(hip_kernels.moment_8bit_bytes(p.numel()), dtype=torch.uint8, device=p.device)
        return torch.zeros_like(p, dtype=torch.promote_types(p.dtype, torch.float32))

    def _first_step(self, p: torch.Tensor) -> Any:
        return torch.zeros((), dtype=torch.float32, device=p.device) if self.capturable else 0

    def _check_param(self, p: torch.Tensor) -> None:
        if not is_dense(p):
            raise ValueError("AdamW needs parameters that fill their memory")
        if self.moment_bits == 8 and p.dtype not in LIST_DTYPES:
            raise ValueError(f"8-bit moments need float32, bfloat16 or float16 parameters, got {p.dtype}")
        if self.moment_bits == 8 and not p.is_contiguous():
            # their bytes say nothing about an order of the dimensions, so a checkpoint could not be checked against it
            raise ValueError("8-bit moments need contiguous parameters")

    def _init_param(self, p: torch.Tensor) -> dict:
        """Makes the state of ``p``, whole or not at all."""
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            # the zeros would be part of the graph and every replay would start from them
            raise RuntimeError("AdamW needs a step before the one that is captured, to make its state")
        self._check_param(p)
        state = {"step": self._first_step(p), "exp_avg": self._moment(p), "exp_avg_sq": self._moment(p)}
        if self.master_weights and p.dtype in (torch.bfloat16, torch.float16):
            state["master"] = p.detach().to(torch.float32)
        held = self.state[p]  # (a dictionary that a caller may hold already)
        held.update(state)
        return held

    @torch.no_grad()
    def _init_group(self, group: dict, skip_non_grad_params: bool = True) -> None:
        """Creates the state of every parameter of ``group`` that does not have one yet."""
        for p in group["params"]:
            if (p.grad is not None or not skip_non_grad_params) and not self.state.get(p):
                self._init_param(p)

    @torch.no_grad()
    def step(self, closure: Optional[Callable[[], float]] = None, *, grad_scale: Optional[torch.Tensor] = None) -> Optional[float]:
        """One optimisation step.  ``closure`` is not supported and must be ``None``.

        ``grad_scale``: one float32 value on the parameters' device that multiplies every gradient, such as the factor
        of ``hip_kernels.global_grad_norm(grads, max_norm=...)``; the gradients themselves stay as they are.
        """
        if closure is not None:
            raise ValueError("closure is not supported")
        capturing = torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()
        if capturing and not self.capturable:
            raise RuntimeError("capturing AdamW.step() needs capturable=True")
        for group in self.param_groups:
            batches: dict = {}
            last = None
            for p in group["params"]:
                grad = p.grad
                if grad is None:
                    continue
                if grad.is_sparse:
                    raise RuntimeError("AdamW does not support sparse gradients")
                state = self.state.get(p) or self._init_param(p)
                key = (p.dtype, grad.dtype, p.get_device(), "master" in state, None if self.capturable else state["step"])
                if key != last:
                    last = key
                    if key not in batches:
                        batches[key] = (self._kernels_take(p, grad), [], [], [])
                    kernels, params, grads, states = batches[key]
                params.append(p)
                grads.append(grad)
                states.append(state)
            for kernels, params, grads, states in batches.values():
                if kernels:
                    self._update_batch(params, grads, states, group, grad_scale)
                    continue
                for p, state in zip(params, states):
                    state["step"] += 1
                    self._update_torch(p, group, grad_scale)
        return None

    @staticmethod
    def _kernels_take(p: torch.Tensor, grad: torch.Tensor) -> bool:
        """Whether the kernels serve the device and the types of ``p`` and its gradient."""
        if not (hip_kernels.on_kernel_device(p) and p.dtype in LIST_DTYPES and grad.dtype in LIST_DTYPES):
            return False
        hip_kernels.require_library()
        return torch.float32 in (p.dtype, grad.dtype) or p.dtype == grad.dtype

    def _update_batch(self, params: list, grads: list, states: list, group: dict, grad_scale: Optional[torch.Tensor]) -> None:
        """One call for parameters of one device, type and step."""
        if not all(map(torch.Tensor.is_contiguous, params)) or not all(map(torch.Tensor.is_contiguous, grads)):
            grads = [g if g.stride() == p.stride() else torch.empty_like(p, dtype=g.dtype).copy_(g) for p, g in zip(params, grads)]
        masters = "master" in states[0]
        update = hip_kernels.fused_adamw_update if self.moment_bits == 32 else hip_kernels.fused_adamw_update_8bit
        rounding = {} if self.moment_bits == 32 else {"rounding": "dithered"}
        steps = [s["step"] for s in states]
        if self.capturable:
            torch._foreach_add_(steps, 1)
        try:
            update(
                [s["master"] for s in states] if masters else params,
                grads,
                [s["exp_avg"] for s in states],
                [s["exp_avg_sq"] for s in states],
                step=steps if self.capturable else steps[0] + 1,
                lr=group["lr"],
                beta1=group["betas"][0],
                beta2=group["betas"][1],
                eps=group["eps"],
                weight_decay=group["weight_decay"],
                weight_decay_method=self.weight_decay_method,
                grad_scale=grad_scale,
                model_params=params if masters else None,
                **rounding,
            )
        except Exception:  # refused before anything was launched: the step does not count
            if self.capturable:
                torch._foreach_sub_(steps, 1)
            raise
        if not self.capturable:
            for state in states:
                state["step"] += 1

    def _update_torch(self, p: torch.Tensor, group: dict, grad_scale: Optional[torch.Tensor]) -> None:
        """The update of one parameter as torch statements, in float32 (float64 parameters: in float64)."""
        state, lr, (beta1, beta2) = self.state[p], group["lr"], group["betas"]
        # a count and a rate on the device stay there (in 64 bits: 1 - beta**t loses its digits in 32), so the statements can
        # be captured
        t = state["step"].double() if self.capturable else state["step"]
        if isinstance(lr, torch.Tensor):
            lr = lr.reshape(()).double() if lr.device == p.device else float(lr)
        held = state.get("master", p)
        wide = torch.promote_types(p.dtype, torch.float32)
        w, grad = held.to(wide, copy=True), p.grad.to(wide, copy=True)
        if grad_scale is not None:
            grad.mul_(grad_scale)
        if isinstance(lr, torch.Tensor) and self.weight_decay_method in ("decoupled", "palm"):
            w.sub_(w * (group["weight_decay"] * (lr if self.weight_decay_method == "decoupled" else lr * lr)))
        else:
            self._apply_weight_decay_inplace(w, grad, lr, group["weight_decay"])
        if self.moment_bits == 8:
            m, v = (_unpack_torch(state[k], p.numel(), k).view(w.shape) for k in ("exp_avg", "exp_avg_sq"))
        else:
            m, v = state["exp_avg"], state["exp_avg_sq"]
        m.lerp_(grad, 1 - beta1)
        v.mul_(beta2).addcmul_(grad, grad, value=1 - beta2)
        den = (v / (1 - beta2**t)).sqrt_().add_(group["eps"])
        w.sub_(lr / (1 - beta1**t) * (m / den))
        if self.moment_bits == 8:
            for k, x in (("exp_avg", m), ("exp_avg_sq", v)):
                state[k].copy_(_pack_torch(x.reshape(-1), k, t))
        held.copy_(w)
        if held is not p:
            p.copy_(w)

    @torch.no_grad()
    def load_state_dict(self, state_dict: dict) -> None:
        """Loads a checkpoint of this class or of ``torch.optim.AdamW``.  Moments come in either width and are held in
        the one of this optimizer; a missing float32 copy of a 16-bit parameter is made from the parameter.  Refuses what
        this class would continue another way: ``maximize``, ``amsgrad``, and ``torch.optim.Adam``'s coupled weight decay
        (unless ``weight_decay_method`` is "l2", which is that).  A refused load changes nothing."""
        before = self.state, self.param_groups
        loaded = state_dict

        def last(_, handed_over: dict) -> None:  # sees what the hooks before the load made of the dictionary
            nonlocal loaded
            loaded = handed_over
            for group in loaded["param_groups"]:
                self._check_loaded_group(group)

        hook = self.register_load_state_dict_pre_hook(last)
        try:
            super().load_state_dict(state_dict)  # (puts new dictionaries in the place of both)
            self._take_states(loaded)
        except BaseException:
            self.state, self.param_groups = before
            raise
        finally:
            hook.remove()

    def _take_states(self, state_dict: dict) -> None:
        """Every loaded state in the widths and types of this optimizer, from the checkpoint itself."""
        saved = state_dict["state"]
        for group, saved_group in zip(self.param_groups, state_dict["param_groups"]):
            for p, index in zip(group["params"], saved_group["params"]):
                if index not in saved:
                    continue
                state = self.state[p]
                self._check_param(p)
                # (the base class casts what it loads to the parameter's type)
                state["exp_avg"], state["exp_avg_sq"] = (self._loaded_moment(saved[index][k], p, k) for k in ("exp_avg", "exp_avg_sq"))
                step = float(saved[index]["step"])
                state["step"] = self._first_step(p).fill_(step) if self.capturable else int(step)
                if self.master_weights and p.dtype in (torch.bfloat16, torch.float16):
                    state["master"] = torch.empty_like(p, dtype=torch.float32).copy_(saved[index].get("master", p.detach()))
                else:
                    state.pop("master", None)

    def _check_loaded_group(self, group: dict) -> None:
        for option in ("maximize", "amsgrad"):
            if group.get(option):
                raise ValueError(f"AdamW cannot continue a checkpoint with {option}=True")
        if not group.get("decoupled_weight_decay", True) and group["weight_decay"] != 0 and self.weight_decay_method != "l2":
            raise ValueError(f'the checkpoint\'s weight decay is not decoupled, which is weight_decay_method="l2" and not "{self.weight_decay_method}"')

    def _loaded_moment(self, value: torch.Tensor, p: torch.Tensor, which: str) -> torch.Tensor:
        """A moment of a checkpoint in the width and the memory order that this optimizer holds it in."""
        packed = value.dtype == torch.uint8 and value.dim() == 1
        if packed and value.numel() != hip_kernels.moment_8bit_bytes(p.numel()) or not packed and value.shape != p.shape:
            raise ValueError(f"{which} of shape {tuple(value.shape)} for a parameter of shape {tuple(p.shape)}")
        if packed == (self.moment_bits == 8):
            return value.to(p.device, copy=True) if packed else self._moment(p).copy_(value)
        kernels = hip_kernels.on_kernel_device(p)
        if packed:
            value, wide = value.to(p.device), torch.empty(p.shape, device=p.device, dtype=torch.float32)
            if kernels:
                hip_kernels.unpack_moments_8bit([value], [wide], which=which)
            else:
                wide.copy_(_unpack_torch(value, p.numel(), which).view(p.shape))
            return self._moment(p).copy_(wide)
        wide, new = value.to(p.device, torch.float32).contiguous(), self._moment(p)
        if kernels:
            hip_kernels.pack_moments_8bit([wide], [new], which=which)
        else:
            new.copy_(_pack_torch(wide.view(-1), which))
        return new
