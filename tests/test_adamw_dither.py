"""8-bit moments of AdamW over many steps: rounding every step to the nearest code would freeze a moving average whose
step is smaller than half the distance between two codes."""

import numpy as np
import pytest
import torch

import _adamw_oracle as O
from emerging_optimizers import hip_kernels as k
from emerging_optimizers.scalar_optimizers import AdamW
from emerging_optimizers.scalar_optimizers.adamw import _pack_torch


def moved(bits, betas, late, steps=8000, change=500, start=2000):
    """How far each weight of the second half of a block moves from step ``start`` on, where that half's gradients are
    ``late`` instead of 1 from step ``change`` on and the first half's stay at 1."""
    p = torch.nn.Parameter(torch.zeros(64))
    opt = AdamW([p], lr=1e-3, betas=betas, weight_decay=0.0, moment_bits=bits)
    p.grad = torch.ones(64)
    for t in range(steps):
        if t == change:
            p.grad[32:] = late
        opt.step()
        if t == start - 1:
            at = p.detach().clone()
    return (p.detach() - at)[32:]


def test_a_moment_without_gradients_decays_to_zero():
    """From the change on the first moment falls by sqrt(0.9) of a code a step.  At code n that is 0.0513 n of a code, and
    a rotation by the golden ratio meets every interval of length d within 2.62 / d steps, so n falls after 51 / n steps
    at most and the sum over n of 51 / n is below 300: long before step 2000 it is 0, and the weights stand still."""
    assert torch.all(moved(32, (0.9, 0.95), 0.0, steps=3000) == 0)
    assert torch.all(moved(8, (0.9, 0.95), 0.0, steps=3000) == 0)


@pytest.mark.parametrize("betas", [(0.9, 0.95), (0.9, 0.999)])
def test_moments_follow_a_fall_of_the_gradients(betas):
    """A tenth of the gradient for half of a block.  The held codes are 40 of 127 and 81 of 255; a dithered code stays
    within one code of the average it follows at the first moment (2/40) and within two at the slower second one
    (2 * 2 / 81 of its root): 10 % of the way at most."""
    wide, narrow = (moved(bits, betas, 0.1) for bits in (32, 8))
    assert torch.all((narrow - wide).abs() <= 0.1 * wide.abs())


def test_dithered_codes_as_torch_statements():
    """The codes are y rounded down or up, by the offset of the step and the place; over a run of steps they average to y."""
    gen = torch.Generator().manual_seed(41)
    x = torch.randn(1000, generator=gen)
    for which, values, unit, power in (("exp_avg", x, 127, 0.5), ("exp_avg_sq", x.square(), 255, 0.25)):
        scale = O.decode(_pack_torch(values, which).numpy(), 1000, which)[1]
        y = unit * (values.abs().double().numpy() / np.repeat(scale, 64)[:1000]) ** power
        total = np.zeros(1000)
        for step in range(5, 1005):
            packed = _pack_torch(values, which, step)
            codes = O.decode(packed.numpy(), 1000, which)[2][:1000]
            assert np.all((abs(codes) >= np.floor(y - 1e-3)) & (abs(codes) <= np.ceil(y + 1e-3))) and abs(codes).max() <= unit
            if which == "exp_avg":
                assert np.all(codes * values.numpy() >= 0)
            assert torch.equal(packed, _pack_torch(values, which, torch.tensor(float(step))))
            total += abs(codes)
        even = y >= (0 if which == "exp_avg" else 6)
        # (a rotation by a quadratic irrational meets an interval its length times n times, off by fewer than 2 + 2 ln n)
        assert np.all(abs(total / 1000 - y)[even] < 0.016 + 1e-4)
        assert np.all((total / 1000 >= y - 1 / 128)[~even])
        for step in (1, 4, torch.tensor(4.0)):
            same = _pack_torch(values, which, step) == _pack_torch(values, which)
            assert float(same.float().mean()) > 0.999


def test_rounding_is_checked():
    with pytest.raises(ValueError, match="rounding must be"):
        k.fused_adamw_update_8bit([], [], [], [], step=1, lr=1e-3, beta1=0.9, beta2=0.95, rounding="up")
    k.fused_adamw_update_8bit([], [], [], [], step=1, lr=1e-3, beta1=0.9, beta2=0.95, rounding="dithered")
