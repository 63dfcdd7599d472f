"""Options of AdamW and arguments of clip_grad_norm_ that are refused, by the constructor and by every group."""

import pytest
import torch

from emerging_optimizers.scalar_optimizers import AdamW
from emerging_optimizers.utils import clip_grad_norm_


def param():
    return torch.nn.Parameter(torch.ones(3))


BAD = [
    (dict(lr=-1e-3), "learning rate"),
    (dict(lr=float("nan")), "learning rate"),
    (dict(betas=(1.0, 0.9)), "betas"),
    (dict(betas=(0.9, -0.1)), "betas"),
    (dict(betas=(float("nan"), 0.9)), "betas"),
    (dict(eps=-1e-8), "eps"),
    (dict(lr=torch.tensor(1e-3)), "capturable"),
]


@pytest.mark.parametrize("options, text", BAD)
def test_bad_options_are_refused_wherever_they_stand(options, text):
    with pytest.raises(ValueError, match=text):
        AdamW([param()], **options)
    with pytest.raises(ValueError, match=text):
        AdamW([dict(params=[param()]), dict(params=[param()], **options)])
    opt = AdamW([param()])
    with pytest.raises(ValueError, match=text):
        opt.add_param_group(dict(params=[param()], **options))
    assert len(opt.param_groups) == 1


def test_good_options_of_groups_are_taken():
    opt = AdamW([dict(params=[param()], lr=0.0, betas=(0.0, 0.5)), dict(params=[param()], eps=0.0)], capturable=True, lr=torch.tensor(0.5))
    assert [g["betas"] for g in opt.param_groups] == [(0.0, 0.5), (0.9, 0.999)]
    with pytest.raises(TypeError):
        opt.add_param_group([param()])
    with pytest.raises(ValueError, match="learning rate"):
        AdamW([param()], capturable=True, lr=torch.tensor(-0.5))


def grads(gen, device="cpu"):
    ps = [torch.nn.Parameter(torch.zeros(7, 3, device=device)), torch.nn.Parameter(torch.zeros(5, device=device))]
    for p in ps:
        p.grad = torch.randn(p.shape, generator=gen).to(device)
    return ps


def test_norm_type_is_an_argument_as_in_torch():
    gen = torch.Generator().manual_seed(61)
    ps = grads(gen)
    raw = [p.grad.clone() for p in ps]
    want = torch.nn.utils.clip_grad_norm_(ps, 0.5, 2.0)
    scaled = [p.grad.clone() for p in ps]
    for norm_type in (2, 2.0):
        for p, g in zip(ps, raw):
            p.grad = g.clone()
        torch.testing.assert_close(clip_grad_norm_(ps, 0.5, norm_type), want, rtol=8 * 2.0**-24, atol=0)
        for p, g in zip(ps, scaled):
            torch.testing.assert_close(p.grad, g, rtol=16 * 2.0**-24, atol=0)
    for norm_type in (1.0, float("inf"), 0):
        with pytest.raises(ValueError, match="norm_type"):
            clip_grad_norm_(ps, 0.5, norm_type)
    with pytest.raises(TypeError):
        clip_grad_norm_(ps, 0.5, 2.0, True)


def test_a_gradient_listed_twice_counts_and_is_scaled_twice():
    gen = torch.Generator().manual_seed(62)
    ps = grads(gen)
    raw = [p.grad.clone() for p in ps]
    norm = clip_grad_norm_([*ps, ps[0]], 0.5)
    exact = float((2 * raw[0].double().square().sum() + raw[1].double().square().sum()).sqrt())
    assert abs(float(norm) - exact) <= 2 * 2.0**-24 * exact
    factor = 0.5 / (exact + 1e-6)
    torch.testing.assert_close(ps[0].grad, raw[0] * factor**2, rtol=16 * 2.0**-24, atol=0)
    torch.testing.assert_close(ps[1].grad, raw[1] * factor, rtol=16 * 2.0**-24, atol=0)
