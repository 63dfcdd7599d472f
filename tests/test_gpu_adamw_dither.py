"""Dithered 8-bit moments on the GPU: codes against their definition in float64, and many steps against 32-bit moments."""

import numpy as np
import pytest
import torch

import _adamw_oracle as O
from emerging_optimizers import hip_kernels as k
from emerging_optimizers.scalar_optimizers import AdamW
from test_gpu_adamw import BF16, F16, F32, HYPER, SIZES, moments, np64, packed_like, snapshot, values

pytestmark = pytest.mark.gpu

ROTATION = {"exp_avg": (0x9E3779B9, 0x6A09E667), "exp_avg_sq": (0x6A09E667, 0xBB67AE85)}


def check_dithered(packed, x, dx, which, step):
    """Every code is floor(y + u) for a value within ``dx`` of ``x``.  y carries the division, root(s) and the product (6 U
    relative), the sums with 1 + u and -1 two roundings of numbers up to 257 (2^-16 each)."""
    n = len(x)
    _, scale, codes = O.decode(packed, n, which)
    assert not codes[n:].any(), "codes behind the last value"
    s = np.repeat(scale, 64)[:n]
    assert np.all(s > 0)
    power, unit = (0.5, 127) if which == "exp_avg" else (0.25, 255)
    by_step, by_place = ROTATION[which]
    u = ((np.arange(n) * by_place + step * by_step & 0xFFFFFFFF) >> 9) * 2.0**-23
    slack = 2.0**-15
    lo = unit * (np.maximum(abs(x) - dx, 0) / s) ** power * (1 - 6 * O.U)
    hi = unit * ((abs(x) + dx) / s) ** power * (1 + 6 * O.U)
    u_lo, u_hi = u, u
    if which == "exp_avg_sq":  # codes below 6 go up; next to 6 either may hold
        u_lo, u_hi = np.where(hi < 6, 255 / 256, u), np.where(lo < 6, np.maximum(u, 255 / 256), u)
        u_lo = np.where(lo < 6, np.minimum(u_lo, 255 / 256), u_lo)
    k_lo, k_hi = np.floor(lo + u_lo - slack), np.minimum(np.floor(hi + u_hi + slack), unit)
    k_lo = np.minimum(k_lo, unit)
    if which == "exp_avg_sq":
        k_lo, k_hi = np.where(x - dx > 0, np.maximum(k_lo, 1), k_lo), np.where(x + dx > 0, np.maximum(k_hi, 1), k_hi)
    size = abs(codes[:n])
    off = (size < k_lo) | (size > k_hi)
    assert not off.any(), f"{off.sum()} of {n} codes off, first at {np.argwhere(off)[0]}"
    if which == "exp_avg":
        c = codes[:n]
        assert np.all((c == 0) | (np.sign(c) == np.sign(x)) | (abs(x) <= dx)), "signs"
    return float(np.mean(k_lo == k_hi))


@pytest.mark.parametrize("types", [(F32, F32, None), (F32, BF16, None), (BF16, BF16, None), (F16, F16, None), (F32, BF16, BF16)], ids=str)
def test_codes_follow_their_definition(gpu, types):
    p_type, g_type, low = types
    gen = torch.Generator().manual_seed(31)
    params, grads = values(gen, SIZES, 0.02, p_type, offset=1), values(gen, SIZES, 1e-3 if g_type != F16 else 1.0, g_type, offset=3)
    ms, vs = moments(gen, SIZES)
    ms, vs = packed_like(ms, "exp_avg"), packed_like(vs, "exp_avg_sq")
    model = None if low is None else values(gen, SIZES, 1.0, low)
    for step in (5, 6, 1000, 100003):
        before = snapshot(params, ms, vs, 8)
        k.fused_adamw_update_8bit(params, grads, ms, vs, step=step, model_params=model, rounding="dithered", **HYPER)
        for i, p in enumerate(params):
            (p2, m2, v2), (dp, dm, dv) = O.adamw(*(x[i] for x in (before[0],)), np64(grads[i]), before[1][i], before[2][i], step=step, method="decoupled", read=8 * O.U, **HYPER)
            O.assert_within(np64(p), p2, O.to_type(p2, dp, p.dtype), f"param {i}")
            if model is not None:
                O.assert_within(np64(model[i]), p2, O.to_type(p2, dp, low), f"copy {i}")
            for packed, x, dx, which in ((ms[i], m2, dm, "exp_avg"), (vs[i], v2, dv, "exp_avg_sq")):
                sure = check_dithered(packed.cpu().numpy(), x, dx, which, step)
                assert len(x) < 1000 or sure > 0.99  # the check leaves no room at nearly all places


def test_first_four_steps_round_to_nearest(gpu):
    gen = torch.Generator().manual_seed(32)
    params, grads = values(gen, SIZES, 0.02), values(gen, SIZES, 1e-3)
    ms, vs = moments(gen, SIZES)
    lists = [[x.clone() for x in params], packed_like(ms, "exp_avg"), packed_like(vs, "exp_avg_sq")]
    other = [[x.clone() for x in part] for part in lists]
    for step in (1, 2, 3, 4, 5):
        k.fused_adamw_update_8bit(lists[0], grads, lists[1], lists[2], step=step, **HYPER)
        k.fused_adamw_update_8bit(other[0], grads, other[1], other[2], step=step, rounding="dithered", **HYPER)
        differ = sum(int((a != b).sum()) for part, twin in zip(lists[1:], other[1:]) for a, b in zip(part, twin))
        total = sum(x.numel() for part in lists[1:] for x in part)
        # (a root that lands on the border between two codes may go either way in another instruction sequence)
        assert differ > 0.2 * total if step == 5 else differ <= 1e-4 * total


def test_step_on_the_device_rotates_as_the_host_number(gpu):
    gen = torch.Generator().manual_seed(33)
    for step in (4, 5, 12345, 1 << 23):
        params, grads = values(gen, SIZES, 0.02), values(gen, SIZES, 1e-3)
        ms, vs = moments(gen, SIZES)
        a = [[x.clone() for x in params], packed_like(ms, "exp_avg"), packed_like(vs, "exp_avg_sq")]
        b = [[x.clone() for x in part] for part in a]
        steps = [torch.tensor(float(step), device=gpu) for _ in params]
        k.fused_adamw_update_8bit(a[0], grads, a[1], a[2], step=step, rounding="dithered", **HYPER)
        k.fused_adamw_update_8bit(b[0], grads, b[1], b[2], step=steps, rounding="dithered", **HYPER)
        for x, y in zip(a[1] + a[2], b[1] + b[2]):
            assert torch.equal(x, y)


@pytest.mark.parametrize("rounding", ["nearest", "dithered"])
def test_a_step_repeats_itself_bit_for_bit(gpu, rounding):
    gen = torch.Generator().manual_seed(34)
    params, grads = values(gen, SIZES, 0.02, BF16), values(gen, SIZES, 1e-3, BF16)
    ms, vs = moments(gen, SIZES)
    start = [params, packed_like(ms, "exp_avg"), packed_like(vs, "exp_avg_sq")]
    runs = []
    for _ in range(3):
        p, m, v = ([x.clone() for x in part] for part in start)
        for step in (7, 8):
            k.fused_adamw_update_8bit(p, grads, m, v, step=step, rounding=rounding, **HYPER)
        runs.append(p + m + v)
    assert all(torch.equal(x, y) for other in runs[1:] for x, y in zip(runs[0], other))


def test_rounding_is_checked(gpu):
    one = [torch.ones(64, device=gpu)]
    packed = [torch.zeros(68, dtype=torch.uint8, device=gpu) for _ in range(2)]
    with pytest.raises(ValueError, match="rounding must be"):
        k.fused_adamw_update_8bit(one, one, packed[:1], packed[1:], step=5, rounding="stochastic", **HYPER)


@pytest.mark.parametrize("betas", [(0.9, 0.95), (0.9, 0.999)])
@pytest.mark.parametrize("late", [0.0, 0.1])
def test_moments_follow_a_change_of_the_gradients(gpu, betas, late):
    """Half of each block's gradients fall to ``late`` after 500 steps, the other half's stay: with gradients of 0 the
    weights stand still from step 2000 on, with 0.1 they go as far as with 32-bit moments, up to one code in 40 of the
    first moment and two codes in 81 of the second one (10 % of the way)."""
    way = []
    for bits in (32, 8):
        p = torch.nn.Parameter(torch.zeros(640, device=gpu))
        opt = AdamW([p], lr=1e-3, betas=betas, weight_decay=0.0, moment_bits=bits)
        p.grad = torch.ones_like(p)
        for t in range(8000 if late else 3000):
            if t == 500:
                p.grad.view(-1, 64)[:, 32:] = late
            opt.step()
            if t == 1999:
                at = p.detach().clone()
        way.append((p.detach() - at).view(-1, 64)[:, 32:])
    if late == 0.0 and betas[1] == 0.95:
        assert torch.all(way[1] == 0)
    if late:
        assert torch.all((way[1] - way[0]).abs() <= 0.1 * way[0].abs())


def test_optimizer_dithers_as_its_cpu_statements(gpu):
    gen = torch.Generator().manual_seed(35)
    p = torch.nn.Parameter((torch.randn(300, 40, generator=gen) * 0.02).to(gpu))
    hyper = dict(lr=1e-2, betas=(0.9, 0.95), weight_decay=0.05, moment_bits=8)
    opt = AdamW([p], **hyper)
    for turn in range(8):
        q = torch.nn.Parameter(p.detach().cpu().clone())
        ref = AdamW([q], **hyper)
        if turn:
            ref.load_state_dict(opt.state_dict())
        g = torch.randn(p.shape, generator=gen)
        p.grad, q.grad = g.to(gpu), g
        opt.step()
        ref.step()
        for key in ("exp_avg", "exp_avg_sq"):
            a, b = opt.state[p][key].cpu()[:12000].to(torch.int16), ref.state[q][key][:12000].to(torch.int16)
            off = ((a - b + 128) % 256 - 128).abs()
            # sums of a few roundings (8 U relative, codes up to 255) move a border by 1.3e-4 of a code at most
            assert int(off.max()) <= 1 and int((off > 0).sum()) <= 12


def test_dithered_steps_replay_from_a_graph(gpu):
    gen = torch.Generator().manual_seed(36)
    start = torch.randn(5000, generator=gen) * 0.02
    ps = [torch.nn.Parameter(start.to(gpu)) for _ in range(2)]
    for p in ps:
        p.grad = torch.zeros_like(p)
    opts = [AdamW([p], lr=torch.tensor(1e-2, device=gpu), betas=(0.9, 0.999), moment_bits=8, capturable=True) for p in ps]
    for opt in opts:
        opt.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opts[0].step()
    for turn in range(12):
        g = torch.randn(5000, generator=gen).to(gpu)
        for p in ps:
            p.grad.copy_(g)
        graph.replay()
        opts[1].step()
        torch.cuda.synchronize()
        assert torch.equal(*ps)
        for key in ("exp_avg", "exp_avg_sq"):
            assert torch.equal(opts[0].state[ps[0]][key], opts[1].state[ps[1]][key])
