"""AdamW, the global norm and the 8-bit moments in float64 numpy, with bounds on what float32 arithmetic may add.

The bounds count roundings.  ``U`` is half a step of float32 relative to the value, the most that one correctly rounded
operation adds; a square root or a quotient may be off by a whole step (2 U) and their combination by 4 U.
"""

import numpy as np
import torch

U = 2.0**-24
HALF_STEP = {torch.float32: U, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
# what rounding to the type adds to values too small for its relative precision (half the smallest number)
TINY = {torch.float32: 2.0**-150, torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25}


def adamw(p, g, m, v, *, step, lr, beta1, beta2, eps, weight_decay, method, scale=1.0, read=0.0):
    """One step in float64: new (p, m, v), and bounds on the error of float32 evaluations of each.  ``read``: relative
    error with which the old moments are read (8 U for the 8-bit form)."""
    p, g, m, v = (np.asarray(x, dtype=np.float64) for x in (p, g, m, v))
    keep = {"decoupled": 1 - lr * weight_decay, "independent": 1 - weight_decay, "palm": 1 - lr * lr * weight_decay, "l2": 1.0}[method]
    l2 = weight_decay if method == "l2" else 0.0
    gs = scale * g + l2 * p
    big_g = abs(scale * g) + abs(l2 * p)  # what rounding of the sum is relative to
    dg = 3 * U * big_g                    # the product, the constant, the sum
    m2 = beta1 * m + (1 - beta1) * gs
    big_m = beta1 * abs(m) + (1 - beta1) * big_g
    dm = (1 - beta1) * dg + beta1 * read * abs(m) + 4 * U * big_m  # two constants, a product, the sum
    v2 = beta2 * v + (1 - beta2) * gs * gs
    dv = (1 - beta2) * (2 * big_g * dg + dg * dg) + beta2 * read * abs(v) + 5 * U * (beta2 * abs(v) + (1 - beta2) * big_g**2)
    c1, c2 = 1 - beta1**step, 1 - beta2**step
    with np.errstate(divide="ignore", invalid="ignore"):
        root = np.sqrt(v2)
        droot = np.where(v2 > 0, np.minimum(dv / np.where(root > 0, root, 1), np.sqrt(dv)), np.sqrt(dv)) + 2 * U * root
        den = root / np.sqrt(c2) + eps
        dden = droot / np.sqrt(c2) + 4 * U * den
        low = np.maximum(den - dden, 1e-300)
        upd = lr / c1 * m2 / den
        dupd = lr / c1 * (dm / low + abs(m2) * dden / (den * low)) + 6 * U * abs(upd)
    p2 = keep * p - upd
    dp = dupd + 2 * U * abs(keep * p) + U * abs(p2)
    return (p2, m2, v2), (dp, dm + 2.0**-149, dv + 2.0**-149)


def to_type(x, bound, dtype):
    """The bound after one more rounding to ``dtype``."""
    return bound + HALF_STEP[dtype] * (abs(x) + bound) + TINY[dtype]


def decode(packed, numel, which):
    """Values of an 8-bit form, block scales and codes, all in float64 / integers."""
    packed = np.asarray(packed)
    blocks = len(packed) // 68
    scale = packed[64 * blocks :].copy().view(np.float32).astype(np.float64)
    raw = packed[: 64 * blocks]
    codes = raw.view(np.int8).astype(np.int64) if which == "exp_avg" else raw.astype(np.int64)
    s = np.repeat(scale, 64)
    with np.errstate(invalid="ignore"):
        value = np.sign(codes) * s * (codes / 127) ** 2 if which == "exp_avg" else s * (codes / 255) ** 4
    return value[:numel], scale, codes


def check_packed(packed, x, dx, which):
    """``packed`` is the 8-bit form of values within ``dx`` of ``x``: every block's scale is its largest magnitude and
    every code one that rounding to nearest may give for some value in the interval."""
    n = len(x)
    _, scale, codes = decode(packed, n, which)
    blocks = len(scale)
    assert blocks == -(-n // 64)
    pad = blocks * 64 - n
    x, dx = np.pad(x, (0, pad)).reshape(blocks, 64), np.pad(dx, (0, pad)).reshape(blocks, 64)
    codes = codes.reshape(blocks, 64)
    assert not codes.reshape(-1)[n:].any(), "codes behind the last value"
    top, least = (abs(x) + dx).max(1), np.maximum(abs(x) - dx, 0).max(1)
    tiny = 2.0**-126
    zero = scale == 0
    assert np.all(least[zero] < tiny), "a block that is not small became 0"
    assert not codes[zero].any()
    assert np.all((scale[~zero] >= least[~zero]) & (scale[~zero] <= top[~zero])), "scales"
    s = np.where(zero, 1.0, scale)[:, None]
    power, unit = (0.5, 127) if which == "exp_avg" else (0.25, 255)
    lo = unit * (np.maximum(abs(x) - dx, 0) / s) ** power
    hi = unit * ((abs(x) + dx) / s) ** power
    # division, root(s) and the product with the unit: at most 6 U relative on the way to the integer
    k_lo = np.ceil(lo * (1 - 6 * U) - 0.5 - 1e-12)
    k_hi = np.floor(np.minimum(hi * (1 + 6 * U), unit) + 0.5 + 1e-12)
    if which == "exp_avg_sq":
        k_lo = np.where(x - dx > 0, np.maximum(k_lo, 1), k_lo)
        k_hi = np.where(x + dx > 0, np.maximum(k_hi, 1), k_hi)
    k = abs(codes)
    ok = ((k >= k_lo) & (k <= k_hi)) | zero[:, None]
    assert ok.all(), f"{(~ok).sum()} codes off, first at {np.argwhere(~ok)[0]}"
    if which == "exp_avg":
        assert np.all((codes == 0) | (np.sign(codes) == np.sign(x)) | (abs(x) <= dx)), "signs"


def assert_within(got, want, bound, what):
    got = np.asarray(got, dtype=np.float64)
    far = abs(got - want) > bound
    assert not far.any(), f"{what}: {far.sum()} of {far.size} values off, worst {np.max(abs(got - want) / bound):.2f} times the bound at {np.argmax(abs(got - want) / bound)}"
