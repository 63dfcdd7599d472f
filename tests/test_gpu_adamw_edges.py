"""Edges of the multi-tensor operators on the GPU: signed zeros and negative values, full argument blocks, memory around
tensors of 16 bits, odd places."""

import numpy as np
import pytest
import torch

import _adamw_oracle as O
from emerging_optimizers import hip_kernels as k
from emerging_optimizers.scalar_optimizers import AdamW
from emerging_optimizers.scalar_optimizers.adamw import _pack_torch
from emerging_optimizers.utils import clip_grad_norm_
from test_gpu_adamw import BF16, F16, F32, HYPER, check_update, moments, np64, packed_like, snapshot, values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_negative_zeros_and_negative_values_in_second_moments(gpu, dtype):
    """Only a value over 0 gets the smallest code at least; -0.0 and a negative value that rounds to 0 get 0."""
    x = torch.zeros(200, dtype=dtype)
    x[0], x[64], x[128] = 2.0, 3.0, 1.0
    x[1:64:2] = -0.0
    x[65:120:3] = -1e-7 if dtype == F16 else -1e-12  # below (0.5 / 255)^4 of 3, the smallest that rounds to code 1, is 4e-11
    x[66:120:3] = 1e-7 if dtype == F16 else 1e-12
    x[130] = -0.5
    packed = packed_like([x.to(gpu)], "exp_avg_sq")[0].cpu()
    codes = packed[:200].to(torch.int64)
    assert not codes[1:64].any()
    if dtype != F16:
        assert not codes[65:120:3].any()
    assert torch.all(codes[66:120:3] >= 1)
    O.check_packed(packed.numpy(), np64(x), np.zeros(200), "exp_avg_sq")
    assert torch.equal(packed, _pack_torch(x.float(), "exp_avg_sq"))


@pytest.mark.parametrize("bits, dtypes", [(32, (torch.float64, torch.float64)), (32, (BF16, F16)), (8, (BF16, F16))], ids=str)
@pytest.mark.parametrize("method", ["decoupled", "l2"])
def test_torch_statements_are_captured_with_tensors(gpu, bits, dtypes, method):
    """Parameters that the kernels do not serve, with a step count and a learning rate on the device: nothing waits for the
    GPU, and replays equal eager steps."""
    p_type, g_type = dtypes
    gen = torch.Generator().manual_seed(52)
    start = torch.randn(100, generator=gen).to(p_type)
    ps = [torch.nn.Parameter(start.to(gpu)) for _ in range(2)]
    opts = [AdamW([p], lr=torch.tensor(0.01, device=gpu), weight_decay=0.1, weight_decay_method=method, moment_bits=bits, capturable=True) for p in ps]
    for p, opt in zip(ps, opts):
        p.grad_dtype = None  # (a gradient of another type than its parameter's)
        p.grad = torch.zeros(100, dtype=g_type, device=gpu)
        opt.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opts[0].step()
    for turn in range(6):
        g = torch.randn(100, generator=gen).to(g_type).to(gpu)
        for p, opt in zip(ps, opts):
            p.grad.copy_(g)
            opt.param_groups[0]["lr"].fill_(0.01 / (turn + 1))
        graph.replay()
        opts[1].step()
        torch.cuda.synchronize()
        assert torch.equal(*ps) and not torch.equal(ps[0].cpu(), start)
        assert float(opts[0].state[ps[0]]["step"]) == turn + 2


@pytest.mark.parametrize("error_if_nonfinite", [False, True])
def test_a_gradient_listed_twice_counts_and_is_scaled_twice(gpu, error_if_nonfinite):
    """As with torch, whose convention clip_grad_norm_ follows; the kernels write no place twice, so such a list goes through
    torch statements."""
    gen = torch.Generator().manual_seed(62)
    ps = [torch.nn.Parameter(torch.zeros(n, device=gpu)) for n in (700, 5)]
    for p in ps:
        p.grad = torch.randn(p.shape, generator=gen).to(gpu)
    raw = [np64(p.grad) for p in ps]
    norm = clip_grad_norm_([*ps, ps[0]], 0.5, error_if_nonfinite=error_if_nonfinite)
    exact = float(np.sqrt(2 * (raw[0] ** 2).sum() + (raw[1] ** 2).sum()))
    assert abs(float(norm) - exact) <= 2 * O.U * exact
    factor = 0.5 / (exact + 1e-6)
    for p, g, f in zip(ps, raw, (factor**2, factor)):
        O.assert_within(np64(p.grad), g * f, 16 * O.U * abs(g * f), "clipped")
