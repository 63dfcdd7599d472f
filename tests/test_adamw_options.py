"""Options of AdamW and arguments of clip_grad_norm_ that are refused, by the constructor and by every group."""

import pytest
import torch

from emerging_optimizers.scalar_optimizers import AdamW


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
