"""Multi-tensor AdamW (moments in 32 and in 8 bits), the global norm and the conversions of 8-bit moments on the GPU,
against the formulas in float64 with bounds that count the roundings of float32 arithmetic (``_adamw_oracle``)."""

import math

import numpy as np
import pytest
import torch

import _adamw_oracle as O
from emerging_optimizers import hip_kernels as k
from emerging_optimizers.orthogonalized_optimizers import Muon
from emerging_optimizers.scalar_optimizers import AdamW
from emerging_optimizers.utils import clip_grad_norm_

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
# one value, short of, at and past the ends of vectors of four, blocks of 64 and chunks of 4096 and of 16384 values
SIZES = [1, 3, 4, 5, 63, 64, 65, 127, 4095, 4096, 4097, 4160, 16383, 16385, 100003]
HYPER = dict(lr=3e-3, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1)


def np64(t):
    return t.detach().float().cpu().numpy().astype(np.float64).reshape(-1)


def values(gen, sizes, scale, dtype=F32, offset=0):
    """Tensors back to back in one buffer, ``offset`` elements behind its start: any alignment occurs."""
    flat = torch.empty(sum(sizes) + offset, dtype=dtype)
    out, at = [], offset
    for n in sizes:
        flat[at : at + n] = (torch.randn(n, generator=gen) * scale * torch.exp(0.5 * torch.randn(n, generator=gen))).to(dtype)
        out.append((at, n))
        at += n
    flat = flat.to("cuda")
    return [flat[a : a + n] for a, n in out]


def moments(gen, sizes, offset=0):
    m = values(gen, sizes, 1e-3, offset=offset)
    v = [x.mul_(x) for x in values(gen, sizes, 1e-3, offset=offset)]
    return m, v


def packed_like(ts, which):
    out = [torch.zeros(k.moment_8bit_bytes(t.numel()), dtype=torch.uint8, device=t.device) for t in ts]
    k.pack_moments_8bit(ts, out, which=which)
    return out


def check_update(params, grads, ms, vs, before, *, method, step, scale=1.0, bits=32, model=None, hyper=HYPER):
    """Every tensor after one update against float64 from the state ``before`` it."""
    p0s, m0s, v0s = before
    for i, p in enumerate(params):
        (p2, m2, v2), (dp, dm, dv) = O.adamw(p0s[i], np64(grads[i]), m0s[i], v0s[i], step=step, method=method, scale=scale, read=0.0 if bits == 32 else 8 * O.U, **hyper)
        O.assert_within(np64(p), p2, O.to_type(p2, dp, p.dtype), f"param {i}")
        if model is not None:
            O.assert_within(np64(model[i]), p2, O.to_type(p2, dp, model[i].dtype), f"copy {i}")
        if bits == 32:
            O.assert_within(np64(ms[i]), m2, dm, f"exp_avg {i}")
            O.assert_within(np64(vs[i]), v2, dv, f"exp_avg_sq {i}")
        else:
            O.check_packed(ms[i].cpu().numpy(), m2, dm, "exp_avg")
            O.check_packed(vs[i].cpu().numpy(), v2, dv, "exp_avg_sq")


def snapshot(params, ms, vs, bits):
    """(p, m, v) in float64.  The kernel reads 8-bit moments with up to 8 roundings of float32, which
    :func:`check_update` adds to the bounds."""
    if bits == 32:
        return [np64(p) for p in params], [np64(m) for m in ms], [np64(v) for v in vs]
    sizes = [p.numel() for p in params]
    return (
        [np64(p) for p in params],
        [O.decode(m.cpu().numpy(), n, "exp_avg")[0] for m, n in zip(ms, sizes)],
        [O.decode(v.cpu().numpy(), n, "exp_avg_sq")[0] for v, n in zip(vs, sizes)],
    )


TYPES = [(F32, F32, None), (F32, BF16, None), (F32, F16, None), (BF16, BF16, None), (BF16, F32, None), (F16, F16, None), (F16, F32, None),
         (F32, BF16, BF16), (F32, F32, BF16), (F32, F16, F16), (F32, F32, F16)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(str(x).replace("torch.", "") for x in t))
def test_update_of_every_type(gpu, types, bits):
    p_type, g_type, low = types
    gen = torch.Generator().manual_seed(1)
    params = values(gen, SIZES, 0.02, p_type, offset=1)
    grads = values(gen, SIZES, 1e-3 if g_type != F16 else 1.0, g_type, offset=3)
    ms, vs = moments(gen, SIZES, offset=2)
    if bits == 8:
        ms, vs = packed_like(ms, "exp_avg"), packed_like(vs, "exp_avg_sq")
    model = None if low is None else values(gen, SIZES, 1.0, low, offset=5)
    update = k.fused_adamw_update if bits == 32 else k.fused_adamw_update_8bit
    for step in (1, 2, 1000):
        before = snapshot(params, ms, vs, bits)
        update(params, grads, ms, vs, step=step, model_params=model, **HYPER)
        check_update(params, grads, ms, vs, before, method="decoupled", step=step, bits=bits, model=model)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("method", ["decoupled", "independent", "l2", "palm"])
def test_update_with_every_decay_method_and_a_gradient_scale(gpu, method, bits):
    gen = torch.Generator().manual_seed(2)
    params, grads = values(gen, SIZES, 0.02), values(gen, SIZES, 1.0)
    ms, vs = moments(gen, SIZES)
    if bits == 8:
        ms, vs = packed_like(ms, "exp_avg"), packed_like(vs, "exp_avg_sq")
    scale = torch.tensor(0.00390625, device=gpu)  # a power of two: its product with the gradient is exact
    kept = [g.clone() for g in grads]
    before = snapshot(params, ms, vs, bits)
    hyper = dict(HYPER, weight_decay=0.01)
    (k.fused_adamw_update if bits == 32 else k.fused_adamw_update_8bit)(
        params, grads, ms, vs, step=7, weight_decay_method=method, grad_scale=scale, **hyper
    )
    check_update(params, grads, ms, vs, before, method=method, step=7, scale=float(scale), bits=bits, hyper=hyper)
    assert all(torch.equal(a, b) for a, b in zip(grads, kept))


@pytest.mark.parametrize("bits", [32, 8])
def test_more_tensors_than_one_launch_takes_and_empty_ones(gpu, bits):
    gen = torch.Generator().manual_seed(3)
    sizes = [0] + [1 + 37 * i % 300 for i in range(150)] + [0, 9000, 0]
    params, grads = values(gen, sizes, 0.02), values(gen, sizes, 1e-3)
    ms, vs = moments(gen, sizes)
    if bits == 8:
        ms, vs = packed_like(ms, "exp_avg"), packed_like(vs, "exp_avg_sq")
    before = snapshot(params, ms, vs, bits)
    (k.fused_adamw_update if bits == 32 else k.fused_adamw_update_8bit)(params, grads, ms, vs, step=3, **HYPER)
    check_update(params, grads, ms, vs, before, method="decoupled", step=3, bits=bits)


@pytest.mark.parametrize("bits", [32, 8])
def test_memory_between_the_tensors_stays_as_it_was(gpu, bits):
    """Weights and gradients with 8 elements of nobody's between them, moments with 64 bytes."""
    gen = torch.Generator().manual_seed(4)
    sizes = [5, 64, 4099, 70]
    ends = np.cumsum([n + 8 for n in sizes]).tolist()
    flats = [torch.full((ends[-1] + 8,), 5.0, device=gpu) for _ in range(4)]
    views = [[f[e - n : e] for e, n in zip(ends, sizes)] for f in flats]
    for vs_, s in zip(views, (0.02, 1e-3, 1e-3, 1e-6)):
        for x in vs_:
            x.copy_(torch.rand(x.shape, generator=gen) * s)
    params, grads, ms, vs = views
    flat8 = None
    if bits == 8:
        lens = [-(-k.moment_8bit_bytes(n) // 16) * 16 for n in sizes]
        at = np.cumsum([0] + [x + 64 for x in lens]).tolist()
        flat8 = [torch.full((at[-1],), 77, dtype=torch.uint8, device=gpu) for _ in range(2)]
        packed = [[f[a : a + k.moment_8bit_bytes(n)] for a, n in zip(at, sizes)] for f in flat8]
        k.pack_moments_8bit(ms, packed[0], which="exp_avg")
        k.pack_moments_8bit(vs, packed[1], which="exp_avg_sq")
        ms, vs = packed
    (k.fused_adamw_update if bits == 32 else k.fused_adamw_update_8bit)(params, grads, ms, vs, step=3, **HYPER)
    norm = k.clip_grads_by_global_norm(grads, max_norm=1e-4)
    assert float(norm) > 1e-4
    for flat in flats:
        for e, n in zip(ends, sizes):
            assert torch.all(flat[e - n - 8 : e - n] == 5.0)
        assert torch.all(flat[ends[-1] :] == 5.0)
    if bits == 8:
        for flat in flat8:
            for a, n in zip(at, sizes):
                assert torch.all(flat[a + k.moment_8bit_bytes(n) : at[at.index(a) + 1]] == 77)


@pytest.mark.parametrize("bits", [32, 8])
def test_step_and_learning_rate_on_the_device_equal_host_numbers(gpu, bits):
    gen = torch.Generator().manual_seed(5)
    for step in (1, 3, 20000):
        params, grads = values(gen, SIZES, 0.02), values(gen, SIZES, 1e-3)
        ms, vs = moments(gen, SIZES)
        if bits == 8:
            ms, vs = packed_like(ms, "exp_avg"), packed_like(vs, "exp_avg_sq")
        before = snapshot(params, ms, vs, bits)
        steps = [torch.tensor(float(step), device=gpu) for _ in params]
        hyper = dict(HYPER, lr=torch.tensor(HYPER["lr"], device=gpu))
        (k.fused_adamw_update if bits == 32 else k.fused_adamw_update_8bit)(params, grads, ms, vs, step=steps, weight_decay_method="palm", **hyper)
        exact = dict(HYPER, lr=float(hyper["lr"]))  # the float32 number
        check_update(params, grads, ms, vs, before, method="palm", step=step, bits=bits, hyper=exact)


@pytest.mark.parametrize("bits", [32, 8])
def test_transposed_parameters_update_in_memory_order(gpu, bits):
    gen = torch.Generator().manual_seed(6)
    p = (torch.randn(70, 130, generator=gen) * 0.02).to(gpu).t()
    g = (torch.randn(70, 130, generator=gen) * 1e-3).to(gpu).t()
    assert not p.is_contiguous()
    m, v = torch.zeros_like(p), torch.zeros_like(p)
    assert m.stride() == p.stride()
    q, h = p.t().contiguous(), g.t().contiguous()
    n, w = torch.zeros_like(q), torch.zeros_like(q)
    if bits == 8:
        m, v, n, w = (torch.zeros(k.moment_8bit_bytes(p.numel()), dtype=torch.uint8, device=gpu) for _ in range(4))
    update = k.fused_adamw_update if bits == 32 else k.fused_adamw_update_8bit
    update([p], [g], [m], [v], step=1, **HYPER)
    update([q], [h], [n], [w], step=1, **HYPER)
    assert torch.equal(p.t(), q)
    with pytest.raises(ValueError, match="order of its param"):
        update([p], [g.contiguous()], [m], [v], step=1, **HYPER)


@pytest.mark.parametrize("bits", [32, 8])
def test_zero_gradients_and_moments_keep_weights_and_nan_stays_in_its_place(gpu, bits):
    p = torch.full((200,), 0.5, device=gpu)
    g = torch.zeros(200, device=gpu)
    m, v = torch.zeros_like(p), torch.zeros_like(p)
    if bits == 8:
        m, v = (torch.zeros(k.moment_8bit_bytes(200), dtype=torch.uint8, device=gpu) for _ in range(2))
    update = k.fused_adamw_update if bits == 32 else k.fused_adamw_update_8bit
    hyper = dict(HYPER, weight_decay=0.0)
    update([p], [g], [m], [v], step=1, **hyper)
    assert torch.all(p == 0.5) and not m.any() and not v.any()
    g[70] = float("nan")
    g[150] = float("inf")
    update([p], [g], [m], [v], step=2, **hyper)
    bad = torch.zeros(200, dtype=torch.bool, device=gpu)
    bad[70] = bad[150] = True
    assert torch.equal(p.isnan(), bad) and torch.all(p[~bad] == 0.5)
    if bits == 8:  # a block shares its scale: the blocks of both become NaN, the others stay 0
        for packed, which in ((m, "exp_avg"), (v, "exp_avg_sq")):
            out = torch.empty(200, device=gpu)
            k.unpack_moments_8bit([packed], [out], which=which)
            assert out[64:192].isnan().all() and not out[:64].any() and not out[192:].any()
    else:
        assert m[70].isnan() and m[150].isinf() and v[150].isinf() and not m[~bad].any()


def test_the_same_memory_twice_and_half_aligned_moments_are_refused(gpu):
    """Refused on the host before any launch; nothing changes."""
    p, g, m, v = (torch.ones(100, device=gpu) for _ in range(4))
    for lists in (([p, p], [g, g], [m, m.clone()], [v, v.clone()]), ([p], [g], [m], [m]), ([p], [p], [m], [v]), ([p[:60], p[50:]], [g[:60], g[50:]], [m[:60], m[50:]], [v[:60], v[50:]])):
        with pytest.raises(ValueError, match="overlaps"):
            k.fused_adamw_update(*lists, step=1, **HYPER)
    with pytest.raises(ValueError, match="overlap"):
        k.clip_grads_by_global_norm([g, g], max_norm=1e-3)
    packed = torch.zeros(2 * 136 + 8, dtype=torch.uint8, device=gpu)
    with pytest.raises(ValueError, match="aligned to 16"):
        k.fused_adamw_update_8bit([p], [g], [packed[8:144]], [packed[144:280]], step=1, **HYPER)
    with pytest.raises(RuntimeError, match="GPU only"):
        k.fused_adamw_update([p], [g], [m], [v.cpu()], step=1, **HYPER)
    with pytest.raises(ValueError, match="grad_scale must be one float32"):
        k.fused_adamw_update([p], [g], [m], [v], step=1, grad_scale=torch.ones(2, device=gpu), **HYPER)
    for t in (p, g, m, v):
        assert torch.all(t == 1)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("shrink", [1.0, 0.25, 1.5e-7, 3e-7])
def test_decay_keeps_the_digits_of_its_share(gpu, bits, shrink):
    """Weights without gradient lose the share ``shrink``, with one rounding of the result, however small the share is
    beside 1 (and all of themselves at 1)."""
    gen = torch.Generator().manual_seed(20)
    p = (torch.randn(5000, generator=gen) * 0.02).to(gpu)
    start = np64(p)
    g = torch.zeros_like(p)
    m, v = torch.zeros_like(p), torch.zeros_like(p)
    if bits == 8:
        m, v = (torch.zeros(k.moment_8bit_bytes(5000), dtype=torch.uint8, device=gpu) for _ in range(2))
    (k.fused_adamw_update if bits == 32 else k.fused_adamw_update_8bit)(
        [p], [g], [m], [v], step=1, **dict(HYPER, weight_decay=shrink), weight_decay_method="independent"
    )
    want = (start - start * float(np.float32(shrink))).astype(np.float32)  # (float64 holds what is rounded to 29 more bits)
    assert np.array_equal(p.cpu().numpy(), want)


def test_extreme_magnitudes_keep_within_float32(gpu):
    """Gradients whose squares underflow leave the update to eps; weights of any size survive."""
    for scale in (1e-30, 1e-20, 1e-10, 1e3, 1e15):
        gen = torch.Generator().manual_seed(7)
        params, grads = values(gen, [1000], 0.02), values(gen, [1000], scale)
        ms, vs = [torch.zeros(1000, device=gpu)], [torch.zeros(1000, device=gpu)]
        before = snapshot(params, ms, vs, 32)
        k.fused_adamw_update(params, grads, ms, vs, step=1, **HYPER)
        if scale >= 1e-15:
            check_update(params, grads, ms, vs, before, method="decoupled", step=1)
        else:  # v is 0 or denormal, sqrt(v) below 1e-16 beside eps = 1e-8
            want = before[0][0] * (1 - HYPER["lr"] * 0.1) - HYPER["lr"] * np64(grads[0]) / 1e-8
            O.assert_within(np64(params[0]), want, 4 * O.U * abs(want) + 1e-10 * abs(HYPER["lr"] * np64(grads[0]) / 1e-8) * 1e3, "param")


# ---------------------------------------------------------------------------------------------
# 8-bit moments
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("which", ["exp_avg", "exp_avg_sq"])
def test_pack_and_unpack(gpu, which, dtype):
    gen = torch.Generator().manual_seed(8)
    sizes = SIZES + [0] + [200] * 140
    x = values(gen, sizes, 1.0, dtype, offset=1)
    if which == "exp_avg_sq":
        x = [t.abs_() for t in x]
    packed = [torch.full((k.moment_8bit_bytes(n),), 255, dtype=torch.uint8, device=gpu) for n in sizes]
    k.pack_moments_8bit(x, packed, which=which)
    for t, q in zip(x, packed):
        O.check_packed(q.cpu().numpy(), np64(t), np.zeros(t.numel()), which)
    for out_type in (F32, BF16, F16):
        out = values(gen, sizes, 1.0, out_type, offset=3)
        k.unpack_moments_8bit(packed, out, which=which)
        for t, q in zip(out, packed):
            want = O.decode(q.cpu().numpy(), t.numel(), which)[0]
            # k^2 times a rounded constant, its square and the scale: the first two roundings count twice
            O.assert_within(np64(t), want, O.to_type(want, 8 * O.U * abs(want), out_type), "unpacked")


@pytest.mark.parametrize("which", ["exp_avg", "exp_avg_sq"])
def test_8bit_form_of_small_scales(gpu, which):
    """Values down to the smallest normal number come back as exactly as large ones (in relative terms, but for what
    float32 itself has no digits for)."""
    gen = torch.Generator().manual_seed(16)
    for scale in (1e-20, 1e-30, 1e-36, 1.2e-38):
        x = torch.rand(64, generator=gen) * scale
        x[5] = scale
        x = x.to(gpu)
        packed, out = packed_like([x], which), torch.empty_like(x)
        k.unpack_moments_8bit(packed, [out], which=which)
        want = O.decode(packed[0].cpu().numpy(), 64, which)[0]
        O.assert_within(np64(out), want, 8 * O.U * abs(want) + 2.0**-149, "unpacked")


def test_blocks_that_are_zero_tiny_or_not_finite(gpu):
    x = torch.zeros(6 * 64 + 10, device=gpu)
    x[64] = 1.1754942e-38     # below the smallest normal number: stored as 0
    x[128] = 1.1754944e-38    # the smallest normal number: kept
    x[192] = float("inf")
    x[256] = float("nan")
    x[320], x[321] = 3.0e38, 1e-30  # a huge and a vanishing value
    x[384] = 2.0
    for which in ("exp_avg", "exp_avg_sq"):
        packed = torch.zeros(k.moment_8bit_bytes(x.numel()), dtype=torch.uint8, device=gpu)
        out = torch.empty_like(x)
        k.pack_moments_8bit([x], [packed], which=which)
        k.unpack_moments_8bit([packed], [out], which=which)
        assert not out[:128].any()
        assert abs(float(out[128]) / 1.1754944e-38 - 1) < 1e-6
        assert out[192:320].isnan().all()
        assert abs(float(out[320]) / 3.0e38 - 1) < 1e-6 and not out[322:384].any()
        # a second moment over 0 keeps the smallest code, a first moment may round to 0
        assert float(out[321]) == 0.0 if which == "exp_avg" else float(out[321]) > 0.0
        assert abs(float(out[384]) - 2.0) < 1e-6
    x = -torch.arange(64, device=gpu, dtype=F32)
    packed = torch.zeros(68, dtype=torch.uint8, device=gpu)
    k.pack_moments_8bit([x], [packed], which="exp_avg")
    O.check_packed(packed.cpu().numpy(), np64(x), np.zeros(64), "exp_avg")


# ---------------------------------------------------------------------------------------------
# norm and clipping
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtypes", [(F32,), (BF16,), (F16,), (F32, BF16, F16)], ids=["f32", "bf16", "f16", "mixed"])
def test_norm_and_clipping(gpu, dtypes):
    gen = torch.Generator().manual_seed(9)
    sizes = [0] + SIZES + [300] * 200 + [70001]
    grads = [values(gen, [n], 0.5, dtypes[i % len(dtypes)], offset=i % 4)[0] for i, n in enumerate(sizes)]
    exact = math.sqrt(sum(float((np64(g) ** 2).sum()) for g in grads))
    before = [np64(g) for g in grads]
    norm, factor = k.global_grad_norm(grads, max_norm=1.5)
    # float64 sums, one rounding to float32; the factor adds a sum, the constants and a quotient
    assert norm.dtype == F32 and norm.shape == () and abs(float(norm) - exact) <= 1.01 * O.U * exact
    want = 1.5 / (exact + 1e-6)
    assert abs(float(factor) - want) <= 6 * O.U * want
    assert float(k.global_grad_norm(grads)) == float(norm)
    assert float(k.global_grad_norm(grads, max_norm=1e9)[1]) == 1.0
    assert float(k.clip_grads_by_global_norm(grads, max_norm=2 * exact)) == float(norm)
    assert all(np.array_equal(np64(g), b) for g, b in zip(grads, before))
    assert float(k.clip_grads_by_global_norm(grads, max_norm=1.5)) == float(norm)
    for g, b in zip(grads, before):
        scaled = b * want
        O.assert_within(np64(g), scaled, O.to_type(scaled, 8 * O.U * abs(scaled), g.dtype) + 1e-300, "scaled")


def test_norm_of_extreme_and_missing_values(gpu):
    big = torch.full((1000,), 3e38, device=gpu)
    assert math.isinf(float(k.global_grad_norm([big])))  # sqrt(1000) 3e38 is past float32
    assert abs(float(k.global_grad_norm([big[:1]])) / 3e38 - 1) < 1e-6  # its square is not, in float64
    small = torch.full((1000,), 1e-30, device=gpu)
    assert abs(float(k.global_grad_norm([small])) / (1e-30 * math.sqrt(1000)) - 1) < 1e-6
    for bad, factor in ((float("inf"), 0.0), (float("nan"), float("nan"))):
        g = torch.ones(5000, device=gpu)
        g[4321] = bad
        norm, f = k.global_grad_norm([g], max_norm=1.0)
        assert not math.isfinite(float(norm))
        assert float(f) == factor or math.isnan(factor) and math.isnan(float(f))
    empty = torch.empty(0, device=gpu)
    norm, f = k.global_grad_norm([empty], max_norm=1.0)
    assert float(norm) == 0.0 and float(f) == 1.0
    assert float(k.clip_grads_by_global_norm([empty, empty], max_norm=0.0)) == 0.0
    assert float(k.global_grad_norm([torch.ones(9, device=gpu)], max_norm=0.0)[1]) == 0.0


def test_norm_is_the_same_every_time(gpu):
    gen = torch.Generator().manual_seed(10)
    grads = values(gen, [1 << 20, 12345, 7], 1.0)
    first = k.global_grad_norm(grads)
    assert all(torch.equal(first, k.global_grad_norm(grads)) for _ in range(5))


def test_a_tensor_of_more_than_two_to_the_33_values(gpu):
    """Offsets past 32 bits, more chunks than one launch takes: slices of a huge bfloat16 tensor that is zero elsewhere,
    against the same slices as tensors of their own."""
    n = (1 << 33) + 4099
    if torch.cuda.mem_get_info()[0] < 90 << 30:
        pytest.skip("needs 90 GiB of free GPU memory")
    gen = torch.Generator().manual_seed(17)
    p, g, out = (torch.zeros(n, dtype=BF16, device=gpu) for _ in range(3))
    packed = [torch.zeros(k.moment_8bit_bytes(n), dtype=torch.uint8, device=gpu) for _ in range(2)]
    places = [slice(a, a + 4096) for a in (0, (1 << 31) - 2048, (1 << 32) - 2048, (1 << 33) - 2048)] + [slice(n - 1987, n)]
    small_p, small_g = [], []
    for place in places:
        p[place] = (torch.randn(place.stop - place.start, generator=gen) * 0.02).to(BF16).to(gpu)
        g[place] = torch.randn(place.stop - place.start, generator=gen).to(BF16).to(gpu)
        small_p.append(p[place].clone())
        small_g.append(g[place].clone())
    norm, factor = k.global_grad_norm([g], max_norm=0.5)
    small_norm, small_factor = k.global_grad_norm(small_g, max_norm=0.5)
    assert abs(float(norm) - float(small_norm)) <= 2 * O.U * float(norm)  # (another order of the float64 sums)
    small = [[torch.zeros(k.moment_8bit_bytes(x.numel()), dtype=torch.uint8, device=gpu) for x in small_p] for _ in range(2)]
    for step in (1, 2):
        k.fused_adamw_update_8bit([p], [g], [packed[0]], [packed[1]], step=step, grad_scale=factor, **HYPER)
        k.fused_adamw_update_8bit(small_p, small_g, *small, step=step, grad_scale=factor, **HYPER)
    for place, want in zip(places, small_p):
        assert torch.equal(p[place], want)
        assert not p[place.stop : place.stop + 64].any() and not p[max(place.start - 64, 0) : place.start].any()
    for mine, theirs, which in zip(packed, small, ("exp_avg", "exp_avg_sq")):
        k.unpack_moments_8bit([mine], [out], which=which)
        for place, q in zip(places, theirs):
            want = torch.empty(place.stop - place.start, dtype=BF16, device=gpu)
            k.unpack_moments_8bit([q], [want], which=which)
            assert torch.equal(out[place], want) and want.any()
            assert not out[place.stop : place.stop + 64].any()
        k.pack_moments_8bit([out], [mine], which=which)
        for place in places:
            again = [torch.empty(k.moment_8bit_bytes(place.stop - place.start), dtype=torch.uint8, device=gpu)]
            k.pack_moments_8bit([out[place]], again, which=which)
            codes = again[0][: place.stop - place.start]
            assert torch.equal(mine[place], codes) and codes.any()
    norm = k.clip_grads_by_global_norm([g], max_norm=0.5)
    k.scale_tensors(small_g, factor)
    for place, want in zip(places, small_g):
        assert torch.equal(g[place], want) and want.any()


# ---------------------------------------------------------------------------------------------
# streams, graphs
# ---------------------------------------------------------------------------------------------
def test_calls_on_two_streams_at_once(gpu):
    """Each call's scratch is its own: norms computed side by side on two streams equal those computed alone."""
    gen = torch.Generator().manual_seed(11)
    lists = [values(gen, [3000000, 77], 1.0), values(gen, [2000000, 99], 3.0)]
    alone = [float(k.global_grad_norm(g)) for g in lists]
    streams = [torch.cuda.Stream() for _ in lists]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for s, g in zip(streams, lists):
            with torch.cuda.stream(s):
                got.append((k.global_grad_norm(g), streams.index(s)))
    torch.cuda.synchronize()
    assert all(float(n) == alone[i] for n, i in got)


@pytest.mark.parametrize("bits", [32, 8])
def test_calls_follow_the_current_stream(gpu, bits):
    """On a side stream, behind work that makes the gradients late: the calls wait for it, as everything on that stream."""
    gen = torch.Generator().manual_seed(18)
    sizes = [100000, 77]
    params, grads = values(gen, sizes, 0.02), values(gen, sizes, 1e-3)
    ms, vs = moments(gen, sizes)
    if bits == 8:
        ms, vs = packed_like(ms, "exp_avg"), packed_like(vs, "exp_avg_sq")
    late = [torch.full_like(g, float("nan")) for g in grads]
    before = snapshot(params, ms, vs, bits)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        for a, b in zip(late, grads):
            a.copy_(b)
        (k.fused_adamw_update if bits == 32 else k.fused_adamw_update_8bit)(params, late, ms, vs, step=4, **HYPER)
        norm = k.clip_grads_by_global_norm(late, max_norm=1e-3)
    side.synchronize()
    check_update(params, grads, ms, vs, before, method="decoupled", step=4, bits=bits)
    exact = math.sqrt(sum(float((np64(g) ** 2).sum()) for g in grads))
    assert abs(float(norm) - exact) <= 1.01 * O.U * exact


def test_two_graphs_replayed_at_once_share_nothing(gpu):
    """Norms of two lists, each in a graph of its own, captured on one stream and replayed side by side on two."""
    gen = torch.Generator().manual_seed(19)
    lists = [values(gen, [4000000, 77], 1.0), values(gen, [3000000, 99], 3.0)]
    graphs, norms = [], []
    k.global_grad_norm(lists[0])
    torch.cuda.synchronize()
    for grads in lists:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norms.append(k.global_grad_norm(grads))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for turn in range(5):
        for grads in lists:
            for g in grads:
                g.mul_(1.5)
        want = [k.global_grad_norm(grads) for grads in lists]
        for n in norms:
            n.zero_()
        torch.cuda.synchronize()
        for _ in range(3):
            for s, graph in zip(streams, graphs):
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(norms, want))


@pytest.mark.parametrize("bits", [32, 8])
def test_clipped_step_replays_from_a_graph(gpu, bits):
    """Norm, factor and update captured once; each replay equals an eager step on the same gradients."""
    gen = torch.Generator().manual_seed(12)
    sizes = [4096, 65, 30001]
    start = [torch.randn(n, generator=gen) * 0.02 for n in sizes]

    def make():
        params = [torch.nn.Parameter(s.to(gpu)) for s in start]
        for p in params:
            p.grad = torch.zeros_like(p)
        return params, AdamW(params, lr=torch.tensor(1e-2, device=gpu), betas=(0.9, 0.95), moment_bits=bits, capturable=True)

    def work(params, opt):
        norm, factor = k.global_grad_norm([p.grad for p in params], max_norm=0.5)
        opt.step(grad_scale=factor)
        return norm

    (a, opt_a), (b, opt_b) = make(), make()
    work(a, opt_a)  # a first step with zero gradients makes the state
    work(b, opt_b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm_a = work(a, opt_a)
    for turn in range(4):
        for p, q in zip(a, b):
            g = (torch.randn(p.shape, generator=gen) * (turn + 1)).to(gpu)
            p.grad.copy_(g)
            q.grad.copy_(g)
        for opt in (opt_a, opt_b):
            opt.param_groups[0]["lr"].fill_(1e-2 / (turn + 1))
        graph.replay()
        norm_b = work(b, opt_b)
        torch.cuda.synchronize()
        assert torch.equal(norm_a, norm_b)
        for p, q in zip(a, b):
            assert torch.equal(p, q)
            assert float(opt_a.state[p]["step"]) == float(opt_b.state[q]["step"]) == turn + 2
            for key in ("exp_avg", "exp_avg_sq"):
                assert torch.equal(opt_a.state[p][key], opt_b.state[q][key])


def test_capture_needs_a_step_count_on_the_device(gpu):
    p = torch.nn.Parameter(torch.ones(10, device=gpu))
    p.grad = torch.ones_like(p)
    opt = AdamW([p])
    opt.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="capturable"):
        with torch.cuda.graph(graph):
            opt.step()


def test_state_is_not_made_inside_a_capture(gpu):
    p = torch.nn.Parameter(torch.ones(10, device=gpu))
    p.grad = torch.ones_like(p)
    opt = AdamW([p], capturable=True)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before the one that is captured"):
        with torch.cuda.graph(graph):
            opt.step()
    assert p not in opt.state or not opt.state[p]
    opt.step()
    assert float(opt.state[p]["step"]) == 1


def test_autograd_notices_what_the_calls_write(gpu):
    """Version counters move with every tensor that a call writes, so a graph that saved one of them refuses to go on."""
    p = torch.nn.Parameter(torch.ones(10, device=gpu))
    loss = (p * p).sum()
    p.grad = torch.ones_like(p)
    m, v, low, grad = torch.zeros_like(p), torch.zeros_like(p), torch.zeros_like(p, dtype=BF16), p.grad
    written = (p, m, v, low)
    before = [t._version for t in written]
    k.fused_adamw_update([p], [grad], [m], [v], step=1, model_params=[low], **HYPER)
    assert all(t._version > b for t, b in zip(written, before))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():  # (tensors without a counter)
        lists = [[torch.ones(10, device=gpu)] for _ in range(4)]
    k.fused_adamw_update(*lists, step=1, **HYPER)
    before = grad._version
    k.global_grad_norm([grad])
    assert grad._version == before
    k.clip_grads_by_global_norm([grad], max_norm=1e-3)
    assert grad._version > before


# ---------------------------------------------------------------------------------------------
# the optimizer
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_uses_the_kernels_and_matches_its_cpu_statements(gpu, bits, master, monkeypatch):
    """Parameters of three types in one optimizer: one call for each kind, and each step's result from the state before
    it, as on the CPU."""
    gen = torch.Generator().manual_seed(13)
    shapes = [((300, 40), F32), ((77,), F32), ((64, 64), BF16), ((33,), F16), ((5, 7, 3), BF16)]
    calls = []
    name = "fused_adamw_update" if bits == 32 else "fused_adamw_update_8bit"
    real = getattr(k, name)
    monkeypatch.setattr(k, name, lambda *a, **kw: (calls.append(len(a[0])), real(*a, **kw)))
    hyper = dict(lr=1e-2, betas=(0.9, 0.95), weight_decay=0.05, weight_decay_method="independent", moment_bits=bits, master_weights=master)
    params = [torch.nn.Parameter((torch.randn(s, generator=gen) * 0.02).to(t).to(gpu)) for s, t in shapes]
    opt = AdamW(params, **hyper)
    for turn in range(3):
        cpu = [torch.nn.Parameter(p.detach().cpu().clone()) for p in params]
        ref = AdamW(cpu, **hyper)
        if turn:
            ref.load_state_dict(opt.state_dict())
        for p, q in zip(params, cpu):
            g = (torch.randn(p.shape, generator=gen)).to(p.dtype)
            p.grad, q.grad = g.to(gpu), g
        calls.clear()
        opt.step()
        ref.step()
        assert sorted(calls) == [1, 2, 2]
        for p, q in zip(params, cpu):
            # float32 evaluations of one step, both within about 20 U of the update and 3 U of the weight, and a rounding
            half = O.HALF_STEP[p.dtype]
            torch.testing.assert_close(p.detach().cpu().float(), q.detach().float(), rtol=2.2 * half, atol=40 * O.U * 1e-2 * 10)
            s, r = opt.state[p], ref.state[q]
            assert s["step"] == r["step"] == turn + 1
            assert ("master" in s) == (master and p.dtype != F32)
            if bits == 32:
                assert s["exp_avg"].dtype == F32
                torch.testing.assert_close(s["exp_avg"].cpu(), r["exp_avg"], rtol=0, atol=20 * O.U * 4)
                torch.testing.assert_close(s["exp_avg_sq"].cpu(), r["exp_avg_sq"], rtol=0, atol=20 * O.U * 16)
            else:
                assert s["exp_avg"].dtype == torch.uint8 and s["exp_avg"].numel() == k.moment_8bit_bytes(p.numel())
                for key in ("exp_avg", "exp_avg_sq"):
                    size = s[key].numel() // 68 * 64
                    a, b = s[key].cpu()[:size].to(torch.int16), r[key][:size].to(torch.int16)
                    assert int(((a - b + 128) % 256 - 128).abs().max()) <= 1  # a code may fall on either side of a border


@pytest.mark.parametrize("capturable", [False, True])
def test_a_refused_step_changes_nothing(gpu, capturable):
    """Two parameters on one piece of memory: the call is refused, steps and moments stay."""
    flat = torch.ones(100, device=gpu)
    a, b = torch.nn.Parameter(flat[:60]), torch.nn.Parameter(flat[50:])
    opt = AdamW([a, b], capturable=capturable)
    a.grad = torch.ones_like(a)
    opt.step()
    kept = flat.clone()
    b.grad = torch.ones_like(b)
    a.grad = a.grad.clone()
    for p in (a, b):
        opt.state[p] = {} if p is b else opt.state[p]
    opt.state[b].update({key: (value.clone() if isinstance(value, torch.Tensor) else value) for key, value in opt.state[a].items()})
    for key in ("exp_avg", "exp_avg_sq"):
        opt.state[b][key] = torch.zeros_like(b)
    with pytest.raises(ValueError, match="overlaps"):
        opt.step()
    assert float(opt.state[a]["step"]) == float(opt.state[b]["step"]) == 1
    assert torch.equal(flat, kept) and not opt.state[b]["exp_avg"].any()


def test_eight_bit_optimizer_follows_the_32_bit_one(gpu):
    """Twenty steps on the same gradients: the 8-bit updates stay within 10 % of the 32-bit ones (each moment is held
    to half a step, at most 1/127 relative for values near the block's largest and more for small ones)."""
    gen = torch.Generator().manual_seed(14)
    start = torch.randn(512, 64, generator=gen) * 0.02
    ps = [torch.nn.Parameter(start.to(gpu)) for _ in range(2)]
    opts = [AdamW([p], lr=1e-3, betas=(0.9, 0.95), weight_decay=0.0, moment_bits=b) for p, b in zip(ps, (32, 8))]
    for _ in range(20):
        g = torch.randn(512, 64, generator=gen).to(gpu)
        for p, opt in zip(ps, opts):
            p.grad = g
            opt.step()
    wide, narrow = (p.detach().cpu() for p in ps)
    assert float((wide - narrow).norm()) < 0.1 * float((wide - start).norm())


def test_checkpoints_between_widths_and_with_torch(gpu):
    gen = torch.Generator().manual_seed(15)
    p = torch.nn.Parameter(torch.randn(100, 30, generator=gen).to(gpu))
    theirs = torch.optim.AdamW([p], lr=1e-3, betas=(0.9, 0.95))
    for _ in range(3):
        p.grad = torch.randn(100, 30, generator=gen).to(gpu)
        theirs.step()
    saved = theirs.state_dict()
    wide = AdamW([p], lr=1e-3, betas=(0.9, 0.95))
    wide.load_state_dict(saved)
    assert wide.state[p]["step"] == 3 and torch.equal(wide.state[p]["exp_avg"], theirs.state[p]["exp_avg"])
    narrow = AdamW([p], lr=1e-3, betas=(0.9, 0.95), moment_bits=8)
    narrow.load_state_dict(wide.state_dict())
    O.check_packed(narrow.state[p]["exp_avg"].cpu().numpy(), np64(wide.state[p]["exp_avg"]), np.zeros(3000), "exp_avg")
    again = AdamW([p], lr=1e-3, betas=(0.9, 0.95), moment_bits=8)
    again.load_state_dict(narrow.state_dict())
    assert torch.equal(again.state[p]["exp_avg_sq"], narrow.state[p]["exp_avg_sq"])
    back = AdamW([p], lr=1e-3, betas=(0.9, 0.95))
    back.load_state_dict(narrow.state_dict())
    want = O.decode(narrow.state[p]["exp_avg_sq"].cpu().numpy(), 3000, "exp_avg_sq")[0]
    O.assert_within(np64(back.state[p]["exp_avg_sq"]), want, 8 * O.U * want + 1e-300, "moment read back")
    turned = torch.nn.Parameter(p.detach().t().contiguous().t())
    other = AdamW([turned], lr=1e-3, betas=(0.9, 0.95))
    other.load_state_dict(narrow.state_dict())
    assert other.state[turned]["exp_avg_sq"].stride() == turned.stride() != p.stride()
    assert torch.equal(other.state[turned]["exp_avg_sq"], back.state[p]["exp_avg_sq"])
    theirs.load_state_dict({**saved, "state": {0: {**wide.state_dict()["state"][0], "step": torch.tensor(3.0)}}})


def test_training_step_with_muon_beside_it(gpu):
    """A small model trained as a user would: backward, clipping over all gradients, Muon for the matrices, AdamW for the
    table, the gains and the head.  Gradients after clipping and the AdamW update are checked against float64."""
    torch.manual_seed(0)
    table = torch.nn.Embedding(50, 64, device=gpu)
    norm = torch.nn.LayerNorm(64, device=gpu)
    hidden = torch.nn.Linear(64, 128, bias=False, device=gpu)
    head = torch.nn.Linear(128, 50, device=gpu)
    rest = [*table.parameters(), *norm.parameters(), *head.parameters()]
    muon = Muon(hidden.parameters(), lr=0.01)
    adamw = AdamW(rest, lr=1e-3, betas=(0.9, 0.95), weight_decay=0.1)
    every = [*rest, *hidden.parameters()]
    ids = torch.randint(0, 50, (4, 16), device=gpu)
    for turn in range(3):
        for p in every:
            p.grad = None
        torch.nn.functional.cross_entropy(head(torch.tanh(hidden(norm(table(ids))))).view(-1, 50), ids.view(-1)).backward()
        raw = [np64(p.grad) for p in every]
        exact = math.sqrt(sum((g**2).sum() for g in raw))
        total = clip_grad_norm_(every, 0.25)
        assert abs(float(total) - exact) <= 1.01 * O.U * exact
        factor = min(1.0, 0.25 / (exact + 1e-6))
        for p, g in zip(every, raw):
            O.assert_within(np64(p.grad), factor * g, 8 * O.U * abs(g) + 1e-300, "clipped gradient")
        zeros = [np.zeros(p.numel()) for p in rest]
        states = [adamw.state[p] for p in rest]
        before = ([np64(p) for p in rest], *([np64(s[key]) for s in states] if turn else zeros for key in ("exp_avg", "exp_avg_sq")))
        weight = hidden.weight.detach().clone()
        muon.step()
        adamw.step()
        assert not torch.equal(weight, hidden.weight)
        check_update(rest, [p.grad for p in rest], [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states], before,
                     method="decoupled", step=turn + 1, hyper=dict(HYPER, lr=1e-3))
