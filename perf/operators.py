"""Cases and plain forms of the multi-tensor optimizer operators.

Four operators act on whole lists of tensors in one call, beside the orthogonalised update of the hidden matrices:

* ``adamw``    one AdamW step, moments held in 32 bits
* ``adamw8``   one AdamW step, moments held in 8 bits with one scale for each block of 64
* ``clip``     the global 2-norm of a list of gradients, and the gradients scaled down to a largest norm
* ``moments``  moments read out of their 8-bit form, and written into it

Each has a plain form in elementary torch operations (used where ``own`` is false) and the calls that a training
program makes of the kernels (where it is true).  A list's tensors are views of one flat buffer, as in a program that
keeps its gradients in buckets; what lies between them belongs to nobody and comes back as it was.
"""

import math
import os
import random
import sys

import torch

own = False

BLOCK = 64  # values that share one scale in the 8-bit form of a moment
_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
BETA1, BETA2, EPS = 0.9, 0.95, 1e-8


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def listed():
    step = {"op": "adamw", "param": "f32", "grad": "f32", "master": False, "clip": False, "decay": "decoupled", "step": 1000, "lr": 1e-4}
    step8 = dict(step, op="adamw8")
    return [
        # the smallest call: the gain of a single normalisation layer, where all of the time is latency
        dict(step, name="adamw one gain", kind="vectors", count=1, width=4096),
        # the gains of a model of 32 layers whose matrices go to the orthogonalised update: two a layer and the last
        dict(step, name="adamw gains", kind="vectors", count=65, width=4096),
        # what such a model leaves to AdamW in full: token table, output head and the gains
        dict(step, name="adamw table and head", kind="table", rows=32768, width=4096, count=65),
        # AdamW for whole layers (4096 wide, 1024 rows of keys and values, 14336 in the feed-forward part) in mixed
        # precision: bf16 weights and gradients, float32 master weights, gradients clipped to a global norm in the step
        dict(step, name="adamw layers, master", kind="layers", count=2, width=4096, kv=1024, ffn=14336, param="bf16", grad="bf16", master=True, clip=True),
        # odd sizes back to back in one bucket, pure bf16, decay in the gradient, the second step of a run
        dict(step, name="adamw odd sizes", kind="odd", count=24, first=777, ratio=1.55, param="bf16", grad="bf16", decay="l2", step=2),
        # the same lists with 8-bit moments: latency, the whole share of AdamW, odd sizes that end inside a block
        dict(step8, name="adamw8 gains", kind="vectors", count=65, width=4096),
        dict(step8, name="adamw8 table and head", kind="table", rows=32768, width=4096, count=65),
        dict(step8, name="adamw8 odd sizes", kind="odd", count=24, first=777, ratio=1.55, param="bf16", grad="bf16", decay="independent", step=2),
        # clipping by the global norm before any optimizer runs: a few small gradients, and all of two layers in bf16
        {"name": "clip gains", "op": "clip", "kind": "vectors", "count": 65, "width": 4096, "grad": "f32"},
        {"name": "clip layers", "op": "clip", "kind": "layers", "count": 2, "width": 4096, "kv": 1024, "ffn": 14336, "grad": "bf16"},
        # 8-bit moments read back in 32 bits, as for a checkpoint that another optimizer continues from
        {"name": "moments read", "op": "moments", "kind": "table", "rows": 32768, "width": 4096, "count": 65, "write": False, "out": "f32"},
        # moments of 32 bits taken over into the 8-bit form, and read back in bf16
        {"name": "moments written", "op": "moments", "kind": "odd", "count": 24, "first": 777, "ratio": 1.55, "write": True, "out": "bf16"},
    ]


def _log_between(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def draw(rng):
    """One more case: another operator, types, number of tensors and sizes, up to a quarter of the largest listed list."""
    op = rng.choice(("adamw", "adamw8", "clip", "moments"))
    case = {"op": op}
    kind = rng.choice(("vectors", "table", "layers", "odd"))
    if kind == "vectors":
        case.update(kind=kind, count=int(_log_between(rng, 1, 400)), width=int(_log_between(rng, 1, 40000)))
    elif kind == "table":
        case.update(kind=kind, rows=int(_log_between(rng, 100, 16384)), width=int(_log_between(rng, 64, 4096)), count=rng.randint(0, 130))
    elif kind == "layers":
        width = 8 * rng.randint(8, 256)
        case.update(kind=kind, count=rng.randint(1, 4), width=width, kv=max(8, width // rng.choice((1, 2, 4, 8))), ffn=int(width * rng.uniform(2, 4)))
    else:
        count = rng.randint(2, 48)
        case.update(kind=kind, count=count, first=int(_log_between(rng, 1, 5000)), ratio=round(rng.uniform(1.0, min(2.0, 1e4 ** (1 / count))), 4))
    if op in ("adamw", "adamw8"):
        param = rng.choice(("f32", "f32", "bf16", "f16"))
        grad = rng.choice(("f32", "bf16", "f16")) if param == "f32" else rng.choice((param, "f32"))
        case.update(param=param, grad=grad, master=param != "f32" and rng.random() < 0.5, clip=rng.random() < 0.5)
        case.update(decay=rng.choice(("decoupled", "independent", "l2", "palm")), step=int(_log_between(rng, 2, 1e5)), lr=1e-4)
    elif op == "clip":
        case.update(grad=rng.choice(("f32", "bf16", "f16")))
    else:
        case.update(write=rng.random() < 0.5, out="bf16")
        if not case["write"]:
            case.update(out=rng.choice(("f32", "bf16")))
    return case


def _shapes(case):
    kind, width = case["kind"], case.get("width")
    if kind == "vectors":
        return [(width,)] * case["count"]
    if kind == "table":
        return [(case["rows"], width)] + [(width,)] * case["count"] + [(case["rows"], width)]
    if kind == "layers":
        kv, ffn = case["kv"], case["ffn"]
        layer = [(width,), (width, width), (kv, width), (kv, width), (width, width), (width,), (ffn, width), (ffn, width), (width, ffn)]
        return layer * case["count"] + [(width,)]
    return [(int(case["first"] * case["ratio"] ** i) | 1,) for i in range(case["count"])]


def work(case):
    n = sum(math.prod(s) for s in _shapes(case))
    grad = n * _BYTES[case.get("grad", "f32")]
    if case["op"] == "clip":
        return {"bytes": 2 * grad, "flops": 3 * n}
    moments8 = 2 * (n + n // 16)  # a byte for each value and four for each block of 64, of both moments
    if case["op"] == "moments":
        read = 8 * n + moments8 if case["write"] else moments8  # 32-bit moments in and their 8-bit form out
        return {"bytes": read + 2 * n * _BYTES[case["out"]], "flops": 12 * n}
    weights = n * (8 + _BYTES[case["param"]]) if case["master"] else n * 2 * _BYTES[case["param"]]
    # 32-bit moments in and out; 8-bit ones in, out and as the bf16 values they stand for
    moments = 16 * n if case["op"] == "adamw" else 2 * moments8 + 4 * n
    return {"bytes": grad + weights + moments, "flops": 15 * n}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _offsets(case):
    """Where each tensor begins in its flat buffer: at multiples of 256 bytes, or back to back for the odd sizes."""
    at, total = [], 0
    for s in _shapes(case):
        at.append(total)
        n = math.prod(s)
        total += n if case["kind"] == "odd" else -(-n // 128) * 128
    return at, total


def _views(flat, case):
    return [flat[a : a + math.prod(s)].view(s) for a, s in zip(_offsets(case)[0], _shapes(case))]


def _flat(case, dtype=torch.float32):
    return torch.zeros(_offsets(case)[1], dtype=dtype, device="cuda")


def _gradient(case, gen):
    """Gradients of a trained model's size; rows of a table whose token did not occur have none."""
    flat = _flat(case)
    scale = torch.exp(0.5 * torch.randn(flat.shape, device="cuda", generator=gen)) * 1e-3
    noise = torch.randn(flat.shape, device="cuda", generator=gen)
    for f, s, z in zip(_views(flat, case), _views(scale, case), _views(noise, case)):
        f.copy_(s * z)
        if case["kind"] == "table" and f.dim() == 2:
            f.mul_(torch.rand(f.shape[0], 1, device="cuda", generator=gen) < 0.7)
    return flat, scale


def _pack_block_form(x, signed):
    """8-bit form of one moment: the codes, then the blocks' float32 scales, as one tensor of bytes."""
    n = x.numel()
    nb = -(-n // BLOCK)
    b = torch.cat([x.reshape(-1).float(), x.new_zeros(nb * BLOCK - n, dtype=torch.float32)]).view(nb, BLOCK)
    codes, scale = _encode(b, signed)
    return torch.cat([codes.reshape(-1).view(torch.uint8), scale.reshape(-1).view(torch.uint8)])


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op, shapes = case["op"], _shapes(case)
    state = {"case": case, "op": op}
    grad, scale = _gradient(case, gen)
    if op == "clip":
        state["grad"] = grad.to(_DTYPES[case["grad"]])
        state["grads"] = _views(state["grad"], case)
        # about half of what the norm of such gradients is: every pass has something to clip
        state["max_norm"] = 0.5e-3 * math.sqrt(sum(math.prod(s) for s in shapes))
        return state
    m32 = 0.3 * scale * torch.randn(scale.shape, device="cuda", generator=gen)
    v32 = scale * scale * torch.exp(0.5 * torch.randn(scale.shape, device="cuda", generator=gen))
    if op == "adamw" or op == "moments" and case["write"]:
        state["exp_avg"], state["exp_avg_sq"] = m32, v32
        state["exp_avgs"], state["exp_avg_sqs"] = _views(m32, case), _views(v32, case)
    if op != "adamw":
        state["exp_avgs8"] = [_pack_block_form(m, True) for m in _views(m32, case)]
        state["exp_avg_sqs8"] = [_pack_block_form(v, False) for v in _views(v32, case)]
        out = _DTYPES[case.get("out", "bf16")]
        state["exp_avg_out"], state["exp_avg_sq_out"] = _flat(case, out), _flat(case, out)
        state["exp_avg_outs"], state["exp_avg_sq_outs"] = _views(state["exp_avg_out"], case), _views(state["exp_avg_sq_out"], case)
        if op == "moments":
            return state
    weights = _flat(case)
    for w in _views(weights, case):
        z = torch.randn(w.shape, device="cuda", generator=gen)
        w.copy_(1.0 + 0.1 * z if w.dim() == 1 and case["kind"] != "odd" else 0.02 * z)
    state["param"] = weights.to(_DTYPES[case["param"]])
    state["params"] = _views(state["param"], case)
    if case["master"]:
        state["master"] = weights
        state["masters"] = _views(weights, case)
    state["grad"] = grad.to(_DTYPES[case["grad"]])
    state["grads"] = _views(state["grad"], case)
    state["step"] = case["step"]
    state["max_norm"] = 0.5e-3 * math.sqrt(sum(math.prod(s) for s in shapes))
    return state


# ---------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------
def _global_norm(grads):
    flat = torch.cat([g.reshape(-1) for g in grads]).float()
    return flat.square().sum(dtype=torch.float64).sqrt().float()


def _clip_factor(norm, max_norm):
    return (max_norm / (norm + 1e-6)).clamp(max=1.0)


def _decay(case, lr):
    """(factor of the weight, multiple of the weight that is added to the gradient)."""
    wd = _weight_decay(case)
    return {"decoupled": (1 - wd * lr, 0.0), "independent": (1 - wd, 0.0), "palm": (1 - wd * lr * lr, 0.0), "l2": (1.0, wd)}[case["decay"]]


def _weight_decay(case):
    """The weight decay that goes with each method: "independent" and "l2" are not multiplied by the learning rate."""
    return {"independent": 1e-5, "l2": 1e-4}.get(case["decay"], 0.1)


def _adamw_plain(state):
    case, lr = state["case"], state["case"]["lr"]
    state["step"] += 1
    factor, l2 = _decay(case, lr)
    out = {}
    gs = [g.float() for g in state["grads"]] if case["grad"] != "f32" else state["grads"]
    if case["clip"]:
        out["norm"] = _global_norm(state["grads"])
        gs = torch._foreach_mul(gs, _clip_factor(out["norm"], state["max_norm"]))
    weights = state["masters"] if case["master"] else state["params"] if case["param"] == "f32" else [p.float() for p in state["params"]]
    if l2:
        gs = torch._foreach_add(gs, weights, alpha=l2)
    ms, vs = state["exp_avgs"], state["exp_avg_sqs"]
    torch._foreach_lerp_(ms, gs, 1 - BETA1)
    torch._foreach_mul_(vs, BETA2)
    torch._foreach_addcmul_(vs, gs, gs, 1 - BETA2)
    den = torch._foreach_sqrt(vs)
    torch._foreach_div_(den, math.sqrt(1 - BETA2 ** state["step"]))
    torch._foreach_add_(den, EPS)
    if factor != 1.0:
        torch._foreach_mul_(weights, factor)
    torch._foreach_addcdiv_(weights, ms, den, -lr / (1 - BETA1 ** state["step"]))
    if case["param"] != "f32":
        torch._foreach_copy_(state["params"], weights)
    out.update(param=state["param"], exp_avg=state["exp_avg"], exp_avg_sq=state["exp_avg_sq"])
    if case["master"]:
        out["master"] = state["master"]
    return out


def _encode(b, signed):
    """Codes and scales of blocks (rows of 64): the first moment as the signed square root of its share of the block's
    largest magnitude, in 127ths; the second, never negative, as the fourth root, in 255ths and never 0 for a value
    over 0.  A block whose largest magnitude is below the smallest normal number is 0, one that holds a value that is not
    finite is NaN throughout."""
    s = b.abs().amax(1, keepdim=True)
    s = torch.where(s.isfinite(), torch.where(s < 2.0**-126, 0.0, s), torch.nan)
    share = torch.where(s > 0, b.abs() / s, 0.0)
    if signed:
        return (share.sqrt() * 127).round().mul(b.sign()).nan_to_num().to(torch.int8), s
    code = (share.sqrt().sqrt() * 255).round()
    return torch.where((b > 0) & (s > 0), code.clamp(min=1), code).nan_to_num().to(torch.uint8), s


def _decode(codes, s, signed):
    c = codes.float()
    if signed:
        return c * c.abs() * (1 / 127**2) * s
    c = c * c * (1 / 255**2)
    return c * c * s


def _blocks(packed, signed):
    """Every tensor's blocks under one another: (codes, scales)."""
    nbs = [p.numel() // (BLOCK + 4) for p in packed]
    codes = torch.cat([p[: BLOCK * nb] for p, nb in zip(packed, nbs)])
    scale = torch.cat([p[BLOCK * nb :] for p, nb in zip(packed, nbs)]).view(torch.float32)
    return (codes.view(torch.int8) if signed else codes).view(-1, BLOCK), scale.view(-1, 1)


def _to_blocks(tensors):
    """Tensors as rows of 64 in 32 bits, each filled up with zeros."""
    zeros = torch.zeros(BLOCK, dtype=tensors[0].dtype, device=tensors[0].device)
    parts = [x for t in tensors for x in (t.reshape(-1), zeros[: -t.numel() % BLOCK])]
    return torch.cat(parts).float().view(-1, BLOCK)


def _from_blocks(b, tensors):
    """The rows' values back into the tensors."""
    sizes = [x for t in tensors for x in (t.numel(), -t.numel() % BLOCK)]
    torch._foreach_copy_([t.view(-1) for t in tensors], list(b.reshape(-1).split(sizes))[::2])


def _store(packed, codes, s):
    nbs = [p.numel() // (BLOCK + 4) for p in packed]
    torch._foreach_copy_([p[: BLOCK * nb] for p, nb in zip(packed, nbs)], list(codes.view(torch.uint8).reshape(-1).split([BLOCK * nb for nb in nbs])))
    torch._foreach_copy_([p[BLOCK * nb :] for p, nb in zip(packed, nbs)], list(s.reshape(-1).view(torch.uint8).split([4 * nb for nb in nbs])))


def _adamw8_plain(state):
    case, lr = state["case"], state["case"]["lr"]
    state["step"] += 1
    factor, l2 = _decay(case, lr)
    out = {}
    g = _to_blocks(state["grads"])
    if case["clip"]:
        out["norm"] = _global_norm(state["grads"])
        g = g * _clip_factor(out["norm"], state["max_norm"])
    held = state["masters"] if case["master"] else state["params"]
    p = _to_blocks(held)
    if l2:
        g = g + l2 * p
    m = _decode(*_blocks(state["exp_avgs8"], True), True)
    v = _decode(*_blocks(state["exp_avg_sqs8"], False), False)
    m = m + (1 - BETA1) * (g - m)
    v = BETA2 * v + (1 - BETA2) * g * g
    den = v.sqrt() / math.sqrt(1 - BETA2 ** state["step"]) + EPS
    p = factor * p - lr / (1 - BETA1 ** state["step"]) * (m / den)
    _from_blocks(p, held)
    if case["master"]:
        _from_blocks(p, state["params"])
        out["master"] = state["master"]
    for x, signed, packed, outs in ((m, True, "exp_avgs8", "exp_avg_outs"), (v, False, "exp_avg_sqs8", "exp_avg_sq_outs")):
        codes, s = _encode(x, signed)
        _store(state[packed], codes, s)
        _from_blocks(_decode(codes, s, signed), state[outs])
    out.update(param=state["param"], exp_avg=state["exp_avg_out"], exp_avg_sq=state["exp_avg_sq_out"])
    return out


def _clip_plain(state):
    # the largest norm falls a little from pass to pass, so that each pass has something to clip
    state["max_norm"] *= 1 - 1e-4
    norm = _global_norm(state["grads"])
    factor = _clip_factor(norm, state["max_norm"])
    gs = [g.float() for g in state["grads"]]
    torch._foreach_mul_(gs, factor)
    torch._foreach_copy_(state["grads"], gs)
    return {"norm": norm, "grad": state["grad"]}


def _moments_plain(state):
    for packed, outs, source, signed in (("exp_avgs8", "exp_avg_outs", "exp_avgs", True), ("exp_avg_sqs8", "exp_avg_sq_outs", "exp_avg_sqs", False)):
        if state["case"]["write"]:
            _store(state[packed], *_encode(_to_blocks(state[source]), signed))
        _from_blocks(_decode(*_blocks(state[packed], signed), signed), state[outs])
    return {"exp_avg": state["exp_avg_out"], "exp_avg_sq": state["exp_avg_sq_out"]}


# ---------------------------------------------------------------------------------------------
# the kernels
# ---------------------------------------------------------------------------------------------
def _kernels():
    """The framework's operators, imported once as a program does."""
    if not hasattr(_kernels, "module"):
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "emerging-optimizers_amd")
        if path not in sys.path:
            sys.path.insert(1, path)
        from emerging_optimizers import hip_kernels

        _kernels.module = hip_kernels
    return _kernels.module


def _adamw_own(state, k):
    case = state["case"]
    state["step"] += 1
    out, factor = {}, None
    if case["clip"]:
        out["norm"], factor = k.global_grad_norm(state["grads"], max_norm=state["max_norm"])
    update = k.fused_adamw_update if state["op"] == "adamw" else k.fused_adamw_update_8bit
    ms, vs = (state["exp_avgs"], state["exp_avg_sqs"]) if state["op"] == "adamw" else (state["exp_avgs8"], state["exp_avg_sqs8"])
    update(
        state["masters"] if case["master"] else state["params"], state["grads"], ms, vs, step=state["step"], lr=case["lr"], beta1=BETA1, beta2=BETA2, eps=EPS,
        weight_decay=_weight_decay(case), weight_decay_method=case["decay"], grad_scale=factor, model_params=state["params"] if case["master"] else None,
    )  # fmt: skip
    if case["master"]:
        out["master"] = state["master"]
    if state["op"] == "adamw":
        out.update(param=state["param"], exp_avg=state["exp_avg"], exp_avg_sq=state["exp_avg_sq"])
        return out
    k.unpack_moments_8bit(ms, state["exp_avg_outs"], which="exp_avg")
    k.unpack_moments_8bit(vs, state["exp_avg_sq_outs"], which="exp_avg_sq")
    out.update(param=state["param"], exp_avg=state["exp_avg_out"], exp_avg_sq=state["exp_avg_sq_out"])
    return out


def _clip_own(state, k):
    state["max_norm"] *= 1 - 1e-4
    norm = k.clip_grads_by_global_norm(state["grads"], max_norm=state["max_norm"])
    return {"norm": norm, "grad": state["grad"]}


def _moments_own(state, k):
    for packed, outs, source, which in (("exp_avgs8", "exp_avg_outs", "exp_avgs", "exp_avg"), ("exp_avg_sqs8", "exp_avg_sq_outs", "exp_avg_sqs", "exp_avg_sq")):
        if state["case"]["write"]:
            k.pack_moments_8bit(state[source], state[packed], which=which)
        k.unpack_moments_8bit(state[packed], state[outs], which=which)
    return {"exp_avg": state["exp_avg_out"], "exp_avg_sq": state["exp_avg_sq_out"]}


def run(state):
    if own:
        return {"adamw": _adamw_own, "adamw8": _adamw_own, "clip": _clip_own, "moments": _moments_own}[state["op"]](state, _kernels())
    return {"adamw": _adamw_plain, "adamw8": _adamw8_plain, "clip": _clip_plain, "moments": _moments_plain}[state["op"]](state)


# ---------------------------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------------------------
def _exact_quantised(x, signed):
    """What a moment is after one trip through 8 bits: for each block of 64 with largest magnitude s, the first moment
    is +-s (k / 127)^2 for the whole k next to 127 sqrt(|x| / s); the second s (k / 255)^4 for the k next to
    255 (x / s)^(1/4), at least 1 for x > 0."""
    n = x.numel()
    rows = torch.nn.functional.pad(x.reshape(-1), (0, -n % BLOCK)).reshape(-1, BLOCK)
    top = rows.abs().max(dim=1, keepdim=True).values
    top = top.masked_fill(top < 2.0**-126, 0.0)
    share = (rows.abs() / top.clamp_min(2.0**-126)).masked_fill(top == 0, 0.0)
    if signed:
        value = torch.sign(rows) * top * (torch.round(127 * share**0.5) / 127) ** 2
    else:
        k = torch.round(255 * share**0.25)
        value = top * (torch.maximum(k, (share > 0).to(k.dtype)) / 255) ** 4
    return value.reshape(-1)[:n].reshape(x.shape)


def _exact_read(packed, shape, signed):
    n = math.prod(shape)
    blocks = packed.numel() // 68
    scale = packed[64 * blocks :].view(torch.float32).double().repeat_interleave(64)[:n]
    code = (packed[: 64 * blocks].view(torch.int8) if signed else packed[: 64 * blocks])[:n].double()
    value = scale * torch.sign(code) * (code / 127) ** 2 if signed else scale * (code / 255) ** 4
    return value.view(shape)


def _exact_norm(grads):
    return math.sqrt(sum(float(g.double().square().sum()) for g in grads))


def _whole(state, key, case, pieces):
    """The flat buffer of 64-bit values that holds the pieces at their places."""
    flat = state[key].double()
    for view, piece in zip(_views(flat, case), pieces):
        view.copy_(piece)
    return flat


def exact(case, seed):
    state = prepare(case, seed)
    shapes = _shapes(case)
    if case["op"] == "moments":
        out = {}
        for name, signed in (("exp_avg", True), ("exp_avg_sq", False)):
            if case["write"]:
                pieces = (_exact_quantised(x.double(), signed) for x in state[name + "s"])
            else:
                pieces = (_exact_read(p, s, signed) for p, s in zip(state[name + "s8"], shapes))
            out[name] = _whole(state, name + "_out", case, pieces)
        return out
    norm = _exact_norm(state["grads"])
    if case["op"] == "clip":
        # the first pass lowers the largest norm before it clips
        factor = min(1.0, state["max_norm"] * (1 - 1e-4) / (norm + 1e-6))
        return {"norm": torch.tensor(norm, dtype=torch.float64), "grad": _whole(state, "grad", case, (factor * g.double() for g in state["grads"]))}
    t, lr, wd = case["step"] + 1, case["lr"], _weight_decay(case)
    factor = min(1.0, state["max_norm"] / (norm + 1e-6)) if case["clip"] else 1.0
    keep = {"decoupled": 1 - lr * wd, "independent": 1 - wd, "palm": 1 - lr * lr * wd, "l2": 1.0}[case["decay"]]
    names = ["exp_avg", "exp_avg_sq", "param"]
    held = state["masters"] if case["master"] else state["params"]
    pieces = {name: [] for name in names}
    whole = {"exp_avg": "exp_avg", "exp_avg_sq": "exp_avg_sq"} if case["op"] == "adamw" else {"exp_avg": "exp_avg_out", "exp_avg_sq": "exp_avg_sq_out"}
    out = {name: state[key].double() for name, key in whole.items()}
    out["param"] = (state["master"] if case["master"] else state["param"]).double()
    places = {name: _views(flat, case) for name, flat in out.items()}
    for i, shape in enumerate(shapes):
        w, g = held[i].double(), factor * state["grads"][i].double()
        if case["decay"] == "l2":
            g = g + wd * w
        if case["op"] == "adamw":
            m, v = state["exp_avgs"][i].double(), state["exp_avg_sqs"][i].double()
        else:
            m, v = _exact_read(state["exp_avgs8"][i], shape, True), _exact_read(state["exp_avg_sqs8"][i], shape, False)
        m = BETA1 * m + (1 - BETA1) * g
        v = BETA2 * v + (1 - BETA2) * g**2
        w = keep * w - lr * (m / (1 - BETA1**t)) / ((v / (1 - BETA2**t)) ** 0.5 + EPS)
        if case["op"] == "adamw8":
            m, v = _exact_quantised(m, True), _exact_quantised(v, False)
        for name, value in (("exp_avg", m), ("exp_avg_sq", v), ("param", w)):
            places[name][i].copy_(value)
    if case["master"]:
        out["master"] = out["param"]
    if case["clip"]:
        out["norm"] = torch.tensor(norm, dtype=torch.float64)
    return out


if __name__ == "__main__":
    print(*(c["name"] for c in listed()), draw(random.Random(0)), sep="\n")
