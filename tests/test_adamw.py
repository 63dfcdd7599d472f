"""Multi-tensor AdamW without a GPU: argument checks of the C entries and of the Python functions, the optimizer's
torch statements against the formulas in float64, 8-bit moments as torch statements, checkpoints, clipping."""

import array
import math

import numpy as np
import pytest
import torch

import _adamw_oracle as O
from emerging_optimizers import _hip
from emerging_optimizers import hip_kernels as k
from emerging_optimizers.scalar_optimizers import AdamW
from emerging_optimizers.scalar_optimizers.adamw import _pack_torch, _unpack_torch
from emerging_optimizers.utils import clip_grad_norm_

HYPER = dict(step=1, lr=1e-3, beta1=0.9, beta2=0.95)


# ---------------------------------------------------------------------------------------------
# C entries: everything is refused before a launch, so made-up addresses do
# ---------------------------------------------------------------------------------------------
_KEPT = []  # arrays live on while a call may read them


def longs(*v):
    _KEPT.append(array.array("q", v))
    return _KEPT[-1]


def at(a):
    return None if a is None else a.buffer_info()[0]


def adamw_rc(p=(1 << 20,), g=(2 << 20,), m=(3 << 20,), v=(4 << 20,), low=None, n=(100,), p_type=0, g_type=0, low_type=1, bits=32, step=1.0,
             lr=1e-3, beta1=0.9, beta2=0.95, eps=1e-8, wd=0.0, method=0, count=None, steps=None):  # fmt: skip
    keep = [longs(*x) if x is not None else None for x in (p, g, m, v, low, steps, n)]
    return _hip.lib().mi_adamw_update(len(n) if count is None else count, *map(at, keep), p_type, g_type, low_type, bits, step, lr, None,
                                      beta1, beta2, eps, wd, method, None, None)  # fmt: skip


@pytest.mark.parametrize(
    "kwargs, code, text",
    [
        (dict(count=-1), _hip.MI_ERR_BAD_ARG, "bad tensor count"),
        (dict(n=(-5,)), _hip.MI_ERR_BAD_ARG, "negative size"),
        (dict(n=((1 << 40) + 1,)), _hip.MI_ERR_UNSUPPORTED_SHAPE, "2\\^40"),
        (dict(p=(0,)), _hip.MI_ERR_BAD_ARG, "param 0 is null"),
        (dict(g=(0,)), _hip.MI_ERR_BAD_ARG, "grad 0 is null"),
        (dict(m=None), _hip.MI_ERR_BAD_ARG, "no list of exp_avg"),
        (dict(p=((1 << 20) + 2,)), _hip.MI_ERR_BAD_ARG, "not aligned to 4"),
        (dict(bits=8, m=((3 << 20) + 8,)), _hip.MI_ERR_BAD_ARG, "not aligned to 16"),
        (dict(p_type=3), _hip.MI_ERR_BAD_ARG, "unknown data type"),
        (dict(p_type=1, g_type=2), _hip.MI_ERR_BAD_ARG, "do not go together"),
        (dict(low=(5 << 20,), low_type=1, g_type=2), _hip.MI_ERR_BAD_ARG, "do not go together"),
        (dict(low=(5 << 20,), low_type=0), _hip.MI_ERR_BAD_ARG, "16-bit copies"),
        (dict(low=(5 << 20,), p_type=1, g_type=1), _hip.MI_ERR_BAD_ARG, "16-bit copies"),
        (dict(bits=16), _hip.MI_ERR_BAD_ARG, "32 or 8 bits"),
        (dict(beta1=1.0), _hip.MI_ERR_BAD_ARG, "betas"),
        (dict(beta2=-0.1), _hip.MI_ERR_BAD_ARG, "betas"),
        (dict(beta2=float("nan")), _hip.MI_ERR_BAD_ARG, "betas"),
        (dict(eps=-1.0), _hip.MI_ERR_BAD_ARG, "eps"),
        (dict(step=0.0), _hip.MI_ERR_BAD_ARG, "step"),
        (dict(steps=(0,)), _hip.MI_ERR_BAD_ARG, "step 0 is null"),
        (dict(method=4), _hip.MI_ERR_BAD_ARG, "decay method"),
        # the same tensor twice, moments over each other, a gradient inside a moment, a copy over its weights
        (dict(p=(1 << 20, 1 << 20), g=(2 << 20, 6 << 20), m=(3 << 20, 7 << 20), v=(4 << 20, 8 << 20), n=(100, 100)), _hip.MI_ERR_BAD_ARG, "overlaps"),
        (dict(v=(3 << 20,)), _hip.MI_ERR_BAD_ARG, "overlaps"),
        (dict(g=((3 << 20) + 396,)), _hip.MI_ERR_BAD_ARG, "overlaps"),
        (dict(low=((1 << 20) + 200,)), _hip.MI_ERR_BAD_ARG, "overlaps"),
        (dict(bits=8, m=(3 << 20,), v=((3 << 20) + 128,)), _hip.MI_ERR_BAD_ARG, "overlaps"),
    ],
)
def test_update_entry_refuses(kwargs, code, text):
    import re

    assert adamw_rc(**kwargs) == code
    assert re.search(text, _hip.last_error()), _hip.last_error()


def test_entries_do_nothing_for_empty_lists():
    lib = _hip.lib()
    assert adamw_rc(p=(), g=(), m=(), v=(), n=()) == _hip.MI_OK
    assert adamw_rc(p=(0,), g=(0,), m=(0,), v=(0,), n=(0,)) == _hip.MI_OK  # (an empty tensor has no address)
    assert lib.mi_scale_tensors(0, None, None, None, 64, None) == _hip.MI_OK
    n = longs(0)
    assert lib.mi_moments_8bit_pack(1, at(n), at(n), at(n), 0, 0, None) == _hip.MI_OK
    assert lib.mi_global_norm_partials_len(0, None) == 0 and lib.mi_global_norm_partials_len(1, at(n)) == 0


def test_norm_scale_and_conversion_entries_refuse():
    lib = _hip.lib()
    x, n, f32, bad = longs(1 << 20, 2 << 20), longs(1000, 1000), array.array("i", [0, 0]), array.array("i", [0, 9])
    need = lib.mi_global_norm_partials_len(2, at(n))
    assert need >= 2
    for args, code, text in (
        ((2, at(x), at(n), at(f32), -1.0, 4096, need, 8192), _hip.MI_ERR_BAD_ARG, "max_norm"),
        ((2, at(x), at(n), at(f32), float("nan"), 4096, need, 8192), _hip.MI_ERR_BAD_ARG, "max_norm"),
        ((2, at(x), at(n), at(f32), 1.0, 4096, need - 1, 8192), _hip.MI_ERR_WORKSPACE, "partial sums"),
        ((2, at(x), at(n), at(f32), 1.0, None, need, 8192), _hip.MI_ERR_WORKSPACE, "partial sums"),
        ((2, at(x), at(n), at(f32), 1.0, 4096, need, None), _hip.MI_ERR_BAD_ARG, "no output"),
        ((2, at(x), at(n), at(bad), 1.0, 4096, need, 8192), _hip.MI_ERR_BAD_ARG, "tensor 1 has an unknown data type"),
        ((2, None, at(n), at(f32), 1.0, 4096, need, 8192), _hip.MI_ERR_BAD_ARG, "no list"),
        ((2, at(longs(1 << 20, 2)), at(n), at(f32), 1.0, 4096, need, 8192), _hip.MI_ERR_BAD_ARG, "tensor 1 is null or not aligned"),
    ):
        for fn in (lib.mi_global_norm, lib.mi_clip_by_global_norm):
            assert fn(*args, None) == code and text in _hip.last_error()
    assert lib.mi_scale_tensors(2, at(x), at(n), at(f32), None, None) == _hip.MI_ERR_BAD_ARG and "no factor" in _hip.last_error()
    same = longs(1 << 20, (1 << 20) + 3996)
    assert lib.mi_scale_tensors(2, at(same), at(n), at(f32), 64, None) == _hip.MI_ERR_BAD_ARG and "overlap" in _hip.last_error()
    assert lib.mi_clip_by_global_norm(2, at(same), at(n), at(f32), 1.0, 4096, need, 8192, None) == _hip.MI_ERR_BAD_ARG and "overlap" in _hip.last_error()
    for fn in (lib.mi_moments_8bit_pack, lib.mi_moments_8bit_unpack):
        assert fn(2, at(x), at(longs(3 << 20, 4 << 20)), at(n), 7, 0, None) == _hip.MI_ERR_BAD_ARG and "data type" in _hip.last_error()
        assert fn(2, at(x), at(longs(3 << 20, 4 << 20)), at(n), 0, 2, None) == _hip.MI_ERR_BAD_ARG and "moment" in _hip.last_error()
        assert fn(2, at(x), at(longs(3 << 20, 1 << 20)), at(n), 0, 0, None) == _hip.MI_ERR_BAD_ARG and "overlaps" in _hip.last_error()
    assert lib.mi_moments_8bit_pack(1, at(x), at(longs((3 << 20) + 4)), at(n), 0, 0, None) == _hip.MI_ERR_BAD_ARG and "16 bytes" in _hip.last_error()


def test_bytes_of_the_8bit_form():
    for n, want in ((0, 0), (1, 68), (64, 68), (65, 136), (1 << 33, (1 << 27) * 68)):
        assert k.moment_8bit_bytes(n) == want == _hip.lib().mi_moment_8bit_bytes(n)


# ---------------------------------------------------------------------------------------------
# Python functions
# ---------------------------------------------------------------------------------------------
def lists(**change):
    out = dict(params=[torch.zeros(4, 6)], grads=[torch.zeros(4, 6)], exp_avgs=[torch.zeros(4, 6)], exp_avg_sqs=[torch.zeros(4, 6)])
    out.update(change)
    return out


@pytest.mark.parametrize(
    "change, exc, text",
    [
        (dict(weight_decay_method="none"), ValueError, "Invalid weight decay method"),
        (dict(grads=[]), TypeError, "grads must have one data type"),
        (dict(grads=[torch.zeros(4, 6)] * 2), ValueError, "2 grads for 1 params"),
        (dict(grads=[torch.zeros(6, 4)]), ValueError, "has shape"),
        (dict(grads=[torch.zeros(6, 4).t()]), ValueError, "order of its param"),
        (dict(params=[torch.zeros(8, 6)[::2]], grads=[torch.zeros(8, 6)[::2]]), ValueError, "must fill its memory"),
        (dict(params=[torch.zeros(4, 6).double()]), TypeError, "params must have one data type"),
        (dict(params=[torch.zeros(4, 6).half(), torch.zeros(4, 6)]), TypeError, "params must have one data type"),
        (dict(exp_avgs=[torch.zeros(4, 6).bfloat16()]), TypeError, "exp_avgs must have one data type"),
        (dict(model_params=[torch.zeros(4, 6)]), TypeError, "model_params must have one data type"),
        (dict(params=[torch.zeros(4, 6).half()], model_params=[torch.zeros(4, 6).half()]), TypeError, "go with float32 params"),
        (dict(), RuntimeError, "GPU only"),
    ],
)
def test_update_function_refuses(change, exc, text):
    with pytest.raises(exc, match=text):
        k.fused_adamw_update(**{**HYPER, **lists(**change)})


def test_update_function_refuses_what_is_not_a_plain_tensor():
    for bad, text in (([1.0], "is not a tensor"), (3, "must be a sequence"), ([torch.zeros(4, 6).to_sparse()], "plain strided"),
                      ([torch.zeros(4, 6, dtype=torch.complex64).conj().imag], "plain strided")):
        with pytest.raises(TypeError, match=text):
            k.fused_adamw_update(**{**HYPER, **lists(grads=bad)})
    with pytest.raises(RuntimeError, match="GPU only"):  # (a step of any number type gets as far as the device)
        k.fused_adamw_update(**{**HYPER, **lists(), "step": np.int64(3)})


def test_a_missing_module_is_an_error(monkeypatch):
    monkeypatch.setattr(_hip, "_lists", None)
    monkeypatch.setattr(_hip, "LISTS_PATH", "/nonexistent/_mi_lists.so")
    with pytest.raises(RuntimeError, match="build it with"):
        k.fused_adamw_update([], [], [], [], **HYPER)


def test_update_functions_take_empty_lists_and_check_packed_moments():
    k.fused_adamw_update([], [], [], [], **HYPER)
    k.fused_adamw_update_8bit([], [], [], [], **HYPER)
    with pytest.raises(TypeError, match="must be uint8"):
        k.fused_adamw_update_8bit(**{**HYPER, **lists()})
    packed = [torch.zeros(67, dtype=torch.uint8)]
    with pytest.raises(ValueError, match="68 contiguous bytes"):
        k.fused_adamw_update_8bit(**{**HYPER, **lists(exp_avgs=packed, exp_avg_sqs=packed)})
    with pytest.raises(ValueError, match="which must be"):
        k.pack_moments_8bit([], [], which="m")
    with pytest.raises(ValueError, match="1 packed for 0"):
        k.unpack_moments_8bit(packed, [], which="exp_avg")
    with pytest.raises(RuntimeError, match="GPU only"):
        k.pack_moments_8bit([torch.zeros(3)], [torch.zeros(68, dtype=torch.uint8)], which="exp_avg")


def test_norm_functions_refuse():
    for fn in (k.global_grad_norm, k.clip_grads_by_global_norm):
        with pytest.raises(ValueError, match="at least one"):
            fn([], max_norm=1.0)
        for bad in (-1.0, float("nan")):
            with pytest.raises(ValueError, match="must not be negative"):
                fn([torch.zeros(3)], max_norm=bad)
        with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
            fn([torch.zeros(3).double()], max_norm=1.0)
        with pytest.raises(ValueError, match="fill their memory"):
            fn([torch.zeros(8)[::2]], max_norm=1.0)
        with pytest.raises(RuntimeError, match="GPU only"):
            fn([torch.zeros(3)], max_norm=1.0)
    k.scale_tensors([], torch.tensor(1.0))
    with pytest.raises(RuntimeError, match="GPU only"):
        k.scale_tensors([torch.zeros(3)], torch.tensor(1.0))


# ---------------------------------------------------------------------------------------------
# the optimizer's torch statements
# ---------------------------------------------------------------------------------------------
def np64(t):
    return t.detach().double().numpy().reshape(-1)


@pytest.mark.parametrize("which", ["exp_avg", "exp_avg_sq"])
def test_8bit_form_as_torch_statements(which):
    for n in (1, 63, 64, 65, 1000):
        x = torch.randn(n) * torch.exp(2 * torch.randn(n))
        x = x if which == "exp_avg" else x.square()
        packed = _pack_torch(x, which)
        assert packed.numel() == k.moment_8bit_bytes(n)
        O.check_packed(packed.numpy(), np64(x), np.zeros(n), which)
        want = O.decode(packed.numpy(), n, which)[0]
        O.assert_within(_unpack_torch(packed, n, which), want, 8 * O.U * abs(want) + 1e-300, "unpacked")


@pytest.mark.parametrize("which", ["exp_avg", "exp_avg_sq"])
def test_8bit_form_of_small_scales_as_torch_statements(which):
    """Values down to the smallest normal number come back as exactly as large ones (in relative terms, but for what
    float32 itself has no digits for)."""
    for scale in (1e-20, 1e-30, 1e-36, 1.2e-38):
        x = torch.rand(64) * scale
        x[5] = scale
        packed = _pack_torch(x, which)
        want = O.decode(packed.numpy(), 64, which)[0]
        O.assert_within(_unpack_torch(packed, 64, which), want, 8 * O.U * abs(want) + 2.0**-149, "unpacked")


def test_oracle_notices_a_wrong_code_scale_and_sign():
    """The checker of 8-bit forms itself: each kind of mistake, planted in a correct form, is found."""
    x = torch.randn(100)
    for which, values in (("exp_avg", x), ("exp_avg_sq", x.square())):
        good = _pack_torch(values, which)
        O.check_packed(good.numpy(), np64(values), np.zeros(100), which)
        for place, change in ((10, 1), (127, 7), (128 + 2, 1)):  # a code, a code behind the end, a scale's bits
            bad = good.clone()
            bad[place] = (int(bad[place]) + change) % 256
            with pytest.raises(AssertionError):
                O.check_packed(bad.numpy(), np64(values), np.zeros(100), which)
    flipped = _pack_torch(-x, "exp_avg")
    with pytest.raises(AssertionError):
        O.check_packed(flipped.numpy(), np64(x), np.zeros(100), "exp_avg")


@pytest.mark.parametrize("method", ["decoupled", "independent", "l2", "palm"])
@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_on_the_cpu_against_float64(bits, method):
    gen = torch.Generator().manual_seed(1)
    p = torch.nn.Parameter(torch.randn(9, 31, generator=gen) * 0.02)
    opt = AdamW([p], lr=1e-2, betas=(0.9, 0.95), weight_decay=0.01, weight_decay_method=method, moment_bits=bits)
    m = v = np.zeros(p.numel())
    for step in (1, 2, 3):
        p.grad = torch.randn(9, 31, generator=gen)
        before = np64(p)
        opt.step(grad_scale=torch.tensor(0.5))
        (p2, m2, v2), (dp, dm, dv) = O.adamw(before, np64(p.grad), m, v, step=step, lr=1e-2, beta1=0.9, beta2=0.95, eps=1e-8,
                                             weight_decay=0.01, method=method, scale=0.5, read=0.0 if bits == 32 else 8 * O.U)  # fmt: skip
        # (the statements round more often than the bounds count: mul, add, lerp and addcmul each, twice as much is allowed)
        O.assert_within(np64(p), p2, 2 * dp, "param")
        s = opt.state[p]
        if bits == 32:
            m, v = np64(s["exp_avg"]), np64(s["exp_avg_sq"])
            O.assert_within(m, m2, 2 * dm, "exp_avg")
            O.assert_within(v, v2, 2 * dv, "exp_avg_sq")
        else:
            O.check_packed(s["exp_avg"].numpy(), m2, 2 * dm, "exp_avg")
            O.check_packed(s["exp_avg_sq"].numpy(), v2, 2 * dv, "exp_avg_sq")
            m, v = (O.decode(s[key].numpy(), p.numel(), key)[0] for key in ("exp_avg", "exp_avg_sq"))


def test_optimizer_equals_torch_adamw_in_float64():
    gen = torch.Generator().manual_seed(2)
    start = torch.randn(5, 7, generator=gen, dtype=torch.float64)
    ps = [torch.nn.Parameter(start.clone()) for _ in range(2)]
    opts = [AdamW([ps[0]], lr=1e-2, betas=(0.8, 0.99), weight_decay=0.1), torch.optim.AdamW([ps[1]], lr=1e-2, betas=(0.8, 0.99), weight_decay=0.1)]
    for _ in range(10):
        g = torch.randn(5, 7, generator=gen, dtype=torch.float64)
        for p, opt in zip(ps, opts):
            p.grad = g.clone()
            opt.step()
    torch.testing.assert_close(ps[0], ps[1], rtol=1e-13, atol=1e-15)
    assert opts[0].state[ps[0]]["exp_avg"].dtype == torch.float64


def test_master_weights_follow_updates_too_small_for_bf16():
    p = torch.nn.Parameter(torch.ones(10, dtype=torch.bfloat16))
    opt = AdamW([p], lr=1e-4, weight_decay=0.0, master_weights=True)
    for _ in range(100):
        p.grad = torch.ones_like(p)
        opt.step()
    assert torch.allclose(opt.state[p]["master"], torch.full((10,), 1 - 100 * 1e-4), rtol=1e-5)
    assert torch.equal(p.detach(), opt.state[p]["master"].bfloat16()) and float(p.detach()[0]) < 1


def test_parameters_without_gradients_keep_their_step_and_state():
    a, b = (torch.nn.Parameter(torch.ones(3)) for _ in range(2))
    opt = AdamW([a, b], weight_decay=0.5)
    a.grad = torch.ones(3)
    opt.step()
    assert b not in opt.state and torch.all(b == 1)
    b.grad = torch.ones(3)
    opt.step()
    assert opt.state[a]["step"] == 2 and opt.state[b]["step"] == 1


def test_optimizer_refuses():
    p = torch.nn.Parameter(torch.ones(4, 4))
    for kwargs, text in (
        (dict(betas=(1.0, 0.9)), "betas"),
        (dict(betas=(0.9, -0.1)), "betas"),
        (dict(eps=-1.0), "eps"),
        (dict(moment_bits=16), "moment_bits"),
        (dict(weight_decay_method="cosine"), "Invalid weight decay method"),
        (dict(lr=torch.tensor(1.0)), "capturable"),
    ):
        with pytest.raises(ValueError, match=text):
            AdamW([p], **kwargs)
    opt = AdamW([p])
    with pytest.raises(ValueError, match="closure"):
        opt.step(lambda: 0.0)
    p.grad = torch.ones(4, 4).to_sparse()
    with pytest.raises(RuntimeError, match="sparse"):
        opt.step()
    q = torch.nn.Parameter(torch.ones(4, 1).expand(4, 4))
    q.grad = torch.ones(4, 4)
    with pytest.raises(ValueError, match="fill their memory"):
        AdamW([q]).step()
    d = torch.nn.Parameter(torch.ones(4, dtype=torch.float64))
    d.grad = torch.ones_like(d)
    with pytest.raises(ValueError, match="8-bit moments"):
        AdamW([d], moment_bits=8).step()


def test_checkpoints_between_widths_and_with_torch_on_the_cpu():
    gen = torch.Generator().manual_seed(3)
    p = torch.nn.Parameter(torch.randn(20, 10, generator=gen).bfloat16())
    theirs = torch.optim.AdamW([p], lr=1e-3)
    p.grad = torch.randn(20, 10, generator=gen).bfloat16()
    theirs.step()
    for master in (False, True):
        wide = AdamW([p], moment_bits=32, master_weights=master)
        wide.load_state_dict(theirs.state_dict())
        s = wide.state[p]
        assert s["step"] == 1 and s["exp_avg"].dtype == torch.float32 and torch.equal(s["exp_avg"], theirs.state[p]["exp_avg"].float())
        assert ("master" in s) is master
        wide.step()
        narrow = AdamW([p], moment_bits=8, master_weights=master)
        narrow.load_state_dict(wide.state_dict())
        n = narrow.state[p]
        assert n["step"] == 2 and n["exp_avg"].dtype == torch.uint8
        O.check_packed(n["exp_avg_sq"].numpy(), np64(s["exp_avg_sq"]), np.zeros(200), "exp_avg_sq")
        if master:
            assert n["master"].dtype == torch.float32 and torch.equal(n["master"], s["master"]) and n["master"] is not s["master"]
        back = AdamW([p], moment_bits=32)
        back.load_state_dict(narrow.state_dict())
        want = O.decode(n["exp_avg"].numpy(), 200, "exp_avg")[0]
        O.assert_within(np64(back.state[p]["exp_avg"]), want, 8 * O.U * abs(want) + 1e-300, "read back")
    capt = AdamW([p], capturable=True)
    capt.load_state_dict(theirs.state_dict())
    assert isinstance(capt.state[p]["step"], torch.Tensor) and float(capt.state[p]["step"]) == 1
    other = torch.nn.Parameter(torch.zeros(300))
    narrow2 = AdamW([other], moment_bits=8)
    saved = narrow.state_dict()
    saved["state"][0].pop("master", None)
    with pytest.raises(ValueError, match="for a parameter of shape"):
        narrow2.load_state_dict(saved)


def test_checkpoints_of_transposed_parameters():
    """Moments are held in the memory order of their parameter, whatever order the checkpoint's have; 8-bit ones say
    nothing about an order and need contiguous parameters."""
    gen = torch.Generator().manual_seed(5)
    a = torch.nn.Parameter(torch.randn(6, 10, generator=gen))
    b = torch.nn.Parameter(a.detach().t().contiguous().t())
    assert not b.is_contiguous()
    opts = [AdamW([p], lr=0.1) for p in (a, b)]
    for turn in range(2):
        g = torch.randn(6, 10, generator=gen)
        for p, opt in zip((a, b), opts):
            p.grad = g.clone()
            opt.step()
        assert torch.equal(a, b)
        opts[1] = AdamW([b], lr=0.1)
        opts[1].load_state_dict(opts[0].state_dict())
        assert opts[1].state[b]["exp_avg"].stride() == b.stride()
    with pytest.raises(ValueError, match="contiguous"):
        AdamW([b], moment_bits=8).step()
    with pytest.raises(ValueError, match="contiguous"):
        AdamW([b], moment_bits=8).load_state_dict(opts[0].state_dict())
    narrow = AdamW([a], lr=0.1, moment_bits=8)
    narrow.load_state_dict(opts[0].state_dict())
    opts[1].load_state_dict(narrow.state_dict())
    want = O.decode(narrow.state[a]["exp_avg"].numpy(), 60, "exp_avg")[0].reshape(6, 10)
    assert opts[1].state[b]["exp_avg"].stride() == b.stride()
    O.assert_within(opts[1].state[b]["exp_avg"].numpy(), want, 8 * O.U * abs(want) + 1e-300, "read back")


def test_clip_grad_norm_on_the_cpu():
    gen = torch.Generator().manual_seed(4)
    ps = [torch.nn.Parameter(torch.zeros(7, 3)), torch.nn.Parameter(torch.zeros(5, dtype=torch.bfloat16)), torch.nn.Parameter(torch.zeros(2))]
    for p in ps[:2]:
        p.grad = torch.randn(p.shape, generator=gen).to(p.dtype)
    raw = [np64(p.grad) for p in ps[:2]]
    exact = math.sqrt(sum((g**2).sum() for g in raw))
    assert abs(float(clip_grad_norm_(ps, 1e9)) - exact) <= 2 * O.U * exact
    assert all(np.array_equal(np64(p.grad), g) for p, g in zip(ps, raw))
    assert abs(float(clip_grad_norm_(iter(ps), 0.5)) - exact) <= 2 * O.U * exact
    f = 0.5 / (exact + 1e-6)
    for p, g in zip(ps, raw):
        O.assert_within(np64(p.grad), f * g, O.to_type(f * g, 8 * O.U * abs(g), p.dtype) + (abs(f * g) * 2.0**-8 if p.dtype == torch.bfloat16 else 0), "clipped")
    assert float(clip_grad_norm_([ps[2]], 1.0)) == 0.0
    with pytest.raises(ValueError, match="negative"):
        clip_grad_norm_(ps, -1.0)
    ps[0].grad[0, 0] = float("nan")
    with pytest.raises(RuntimeError, match="global 2-norm"):
        clip_grad_norm_(ps, 1.0, error_if_nonfinite=True)
