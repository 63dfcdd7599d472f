"""Checkpoints and copies of AdamW: what cannot be continued is refused before anything changes, what can be is whole."""

import copy
import pickle

import pytest
import torch

from emerging_optimizers.scalar_optimizers import AdamW


def stepped(cls=AdamW, shape=(6,), dtype=torch.float32, **kwargs):
    """An optimizer of one parameter after one step, and the parameter."""
    p = torch.nn.Parameter(torch.linspace(-1, 1, 6).reshape(shape).to(dtype))
    opt = cls([p], **kwargs)
    p.grad = torch.linspace(0.5, 1.5, 6).reshape(shape).to(dtype)
    opt.step()
    return opt, p


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize(
    "cls, options, text",
    [
        (torch.optim.AdamW, dict(maximize=True), "maximize"),
        (torch.optim.AdamW, dict(amsgrad=True), "amsgrad"),
        (torch.optim.Adam, dict(weight_decay=0.1), "decoupled"),
    ],
)
def test_checkpoints_of_another_rule_are_refused(cls, options, text, bits):
    """Gradients followed upwards, the running maximum of second moments, decay that goes through the moments: a step of
    this class would go another way than the run that is continued."""
    theirs, _ = stepped(cls, lr=0.1, **options)
    mine, p = stepped(lr=0.3, moment_bits=bits)
    before = copy.deepcopy(mine.state_dict())
    with pytest.raises(ValueError, match=text):
        mine.load_state_dict(theirs.state_dict())
    after = mine.state_dict()
    assert after["param_groups"] == before["param_groups"]
    assert all(torch.equal(torch.as_tensor(a), torch.as_tensor(b)) for a, b in zip(after["state"][0].values(), before["state"][0].values()))


def test_checkpoints_of_the_same_rule_load():
    for cls, options in ((torch.optim.AdamW, dict(weight_decay=0.1)), (torch.optim.Adam, dict(weight_decay=0.0))):
        theirs, p = stepped(cls, lr=0.1, **options)
        q = torch.nn.Parameter(p.detach().clone())
        mine = AdamW([q], lr=0.3)
        mine.load_state_dict(theirs.state_dict())
        q.grad = p.grad
        for opt in (theirs, mine):
            opt.step()
        # each side rounds its moments, the quotient and the weight: about 10 roundings of an update of 0.1
        torch.testing.assert_close(q, p, rtol=2 * 2.0**-24, atol=10 * 0.1 * 2.0**-24)
    theirs, p = stepped(torch.optim.Adam, lr=0.1, weight_decay=0.1)
    AdamW([p], weight_decay_method="l2").load_state_dict(theirs.state_dict())


def same(a, b):
    """Whether two state dictionaries hold the same."""
    if isinstance(a, dict):
        return isinstance(b, dict) and a.keys() == b.keys() and all(same(a[key], b[key]) for key in a)
    if isinstance(a, (list, tuple)):
        return len(a) == len(b) and all(map(same, a, b))
    if isinstance(a, torch.Tensor):
        return isinstance(b, torch.Tensor) and a.dtype == b.dtype and torch.equal(a, b)
    return a == b


@pytest.mark.parametrize("how, bits", [(how, bits) for how in ("shape", "packed size", "missing moment") for bits in (32, 8)] + [("transposed parameter", 8)])
def test_a_refused_load_changes_nothing(how, bits):
    """Whatever is wrong with the second of two parameters' states, the optimizer goes on as if nothing had been loaded."""

    def make(lr):
        ps = [torch.nn.Parameter(torch.linspace(-1, 1, 70).bfloat16()), torch.nn.Parameter(torch.linspace(0, 1, 12).view(3, 4).bfloat16())]
        opt = AdamW(ps, lr=lr, moment_bits=bits)
        for p in ps:
            p.grad = torch.ones_like(p)
        opt.step()
        return opt, ps

    saved, (mine, ps) = make(0.5)[0].state_dict(), make(0.1)
    bad = saved["state"][1]
    if how == "shape":
        bad["exp_avg_sq"] = torch.zeros(4, 3)
    elif how == "packed size":
        bad["exp_avg"] = torch.zeros(136, dtype=torch.uint8)
    elif how == "missing moment":
        del bad["exp_avg"]
    else:
        ps[1].data = ps[1].data.t().contiguous().t()
    before = copy.deepcopy(mine.state_dict())
    with pytest.raises((ValueError, KeyError)):
        mine.load_state_dict(saved)
    assert same(mine.state_dict(), before)
    if how != "transposed parameter":
        mine.step()
        assert mine.state[ps[0]]["step"] == 2


def test_load_hooks_see_and_change_what_is_loaded():
    """A hook before the load may hand over another dictionary: its moments are taken, not the caller's."""
    theirs, p = stepped(lr=0.1)
    saved = theirs.state_dict()
    renamed = {"state": {0: {"step": 1, "m": saved["state"][0]["exp_avg"], "v": saved["state"][0]["exp_avg_sq"]}}, "param_groups": saved["param_groups"]}

    def names(opt, loaded):
        state = {i: {"step": s["step"], "exp_avg": s["m"] * 2, "exp_avg_sq": s["v"]} for i, s in loaded["state"].items()}
        return {**loaded, "state": state}

    mine = AdamW([p], lr=0.3)
    handle = mine.register_load_state_dict_pre_hook(names)
    mine.load_state_dict(renamed)
    assert torch.equal(mine.state[p]["exp_avg"], 2 * saved["state"][0]["exp_avg"]) and mine.param_groups[0]["lr"] == 0.1
    handle.remove()
    mine.load_state_dict(saved)
    assert torch.equal(mine.state[p]["exp_avg"], saved["state"][0]["exp_avg"])
    upwards = copy.deepcopy(saved)
    mine.register_load_state_dict_pre_hook(lambda opt, loaded: {**upwards, "param_groups": [{**upwards["param_groups"][0], "maximize": True}]})
    with pytest.raises(ValueError, match="maximize"):
        mine.load_state_dict(saved)
    assert len(mine._optimizer_load_state_dict_pre_hooks) == 1


def test_a_refused_first_step_leaves_no_state():
    p = torch.nn.Parameter(torch.ones(4, 1).expand(4, 4))
    p.grad = torch.ones(4, 4)
    opt = AdamW([p])
    for call in (opt.step, lambda: opt._init_group(opt.param_groups[0])):
        with pytest.raises(ValueError, match="fill their memory"):
            call()
        assert p not in opt.state
    q = torch.nn.Parameter(torch.ones(4, 4))
    AdamW([q]).load_state_dict(opt.state_dict())
    q.grad = torch.ones(4, 4)
    opt = AdamW([q])
    held = opt.state[q]
    opt.step()
    assert held is opt.state[q] and held["step"] == 1


@pytest.mark.parametrize("make", [copy.deepcopy, lambda opt: pickle.loads(pickle.dumps(opt))], ids=["deepcopy", "pickle"])
@pytest.mark.parametrize(
    "options", [dict(), dict(moment_bits=8, weight_decay_method="independent"), dict(master_weights=True, weight_decay_method="palm"), dict(capturable=True)]
)
def test_copies_go_on_as_the_original(make, options):
    opt, p = stepped(dtype=torch.bfloat16, lr=0.1, **options)
    twin = make(opt)
    q = twin.param_groups[0]["params"][0]
    assert q is not p and torch.equal(q, p)
    for _ in range(3):
        p.grad = torch.linspace(-1, 1, 6).bfloat16()
        q.grad = p.grad.clone()
        opt.step()
        twin.step()
    assert torch.equal(q, p) and same(opt.state_dict(), twin.state_dict())
