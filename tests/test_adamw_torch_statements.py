"""AdamW's torch statements (other devices and types than the kernels serve): counters and learning rates in tensors."""

import pytest
import torch

from emerging_optimizers.scalar_optimizers import AdamW


@pytest.mark.parametrize("method", ["decoupled", "independent", "l2", "palm"])
@pytest.mark.parametrize("betas", [(0.9, 0.999), (0.0, 0.0), (0.9999, 0.99999)])
def test_float64_with_tensors_equals_numbers(betas, method):
    """1 - beta**t loses its digits in float32 for small t; float64 parameters get float64 results either way.  The two
    sides take the same statements but for the order of the decay: a few roundings of 1.1e-16."""
    gen = torch.Generator().manual_seed(51)
    start = torch.randn(20, generator=gen, dtype=torch.float64)
    ps = [torch.nn.Parameter(start.clone()) for _ in range(2)]
    lr = 0.125  # the same number in float32
    options = dict(betas=betas, weight_decay=0.1, weight_decay_method=method)
    opts = [AdamW([ps[0]], lr=lr, **options), AdamW([ps[1]], lr=torch.tensor(lr), capturable=True, **options)]
    for _ in range(5):
        g = torch.randn(20, generator=gen, dtype=torch.float64)
        for p, opt in zip(ps, opts):
            p.grad = g.clone()
            opt.step()
        torch.testing.assert_close(ps[1], ps[0], rtol=1e-12, atol=1e-14)
    assert opts[1].param_groups[0]["lr"].dtype == torch.float32 and float(opts[1].state[ps[1]]["step"]) == 5
