"""AdamW.load_state_dict: options of another optimizer's groups that this step
does not follow are refused before anything changes."""
import copy

import pytest
import torch

from ceo_firm_matching import AdamW


def stepped(opt_class, steps=2, **kw):
    torch.manual_seed(0)
    p = torch.nn.Parameter(torch.linspace(-1, 1, 130))
    opt = opt_class([p], lr=1e-2, **kw)
    for _ in range(steps):
        p.grad = torch.randn(130)
        opt.step()
    return p, opt


def snapshot(opt):
    g = {k: v for k, v in opt.param_groups[0].items() if k != "params"}
    return copy.deepcopy(g), [x.clone() for x in opt.held_states()], int(opt.state[opt.param_groups[0]["params"][0]]["step"])


def unchanged(opt, before):
    after = snapshot(opt)
    return after[0] == before[0] and all(torch.equal(a, b) for a, b in zip(after[1], before[1])) and after[2] == before[2]


@pytest.mark.parametrize("steps", [0, 2])
@pytest.mark.parametrize("option", ["maximize", "amsgrad"])
def test_torch_options_that_change_the_step(option, steps):
    _, theirs = stepped(torch.optim.AdamW, steps, **{option: True})
    _, opt = stepped(AdamW)
    before = snapshot(opt)
    with pytest.raises(NotImplementedError, match=option):
        opt.load_state_dict(theirs.state_dict())
    assert unchanged(opt, before)
    sd = copy.deepcopy(stepped(AdamW)[1].state_dict())
    sd["param_groups"][0]["differentiable"] = True
    with pytest.raises(NotImplementedError, match="differentiable"):
        opt.load_state_dict(sd)
    assert unchanged(opt, before)
    with pytest.raises(NotImplementedError, match=option):
        AdamW([{"params": [torch.nn.Parameter(torch.ones(3))], option: True}])


def test_decay_that_is_not_decoupled():
    """torch.optim.Adam adds its decay to the gradient: its states load where it has none."""
    _, opt = stepped(AdamW)
    before = snapshot(opt)
    with pytest.raises(NotImplementedError, match="decay"):
        opt.load_state_dict(stepped(torch.optim.Adam, weight_decay=0.1)[1].state_dict())
    assert unchanged(opt, before)
    p, theirs = stepped(torch.optim.Adam)
    q, opt = stepped(AdamW)
    opt.load_state_dict(theirs.state_dict())
    with torch.no_grad():
        q.copy_(p)
    p.grad = q.grad = torch.full((130,), 0.5)
    theirs.step()
    opt.step()
    # one step of at most lr; values <= 2, each side rounds a few times
    assert float((p - q).detach().abs().max()) <= 8 * 2.0 ** -24 * 2


@pytest.mark.parametrize("key,value", [("lr", -1e-3), ("lr", float("inf")), ("betas", (0.9, 1.0)), ("eps", -1.0), ("eps", float("inf")),
                                       ("weight_decay", -0.1), ("weight_decay", float("nan"))])
def test_loaded_hyperparameters_are_checked(key, value):
    _, opt = stepped(AdamW)
    before = snapshot(opt)
    sd = copy.deepcopy(stepped(AdamW, 1)[1].state_dict())
    sd["param_groups"][0][key] = value
    with pytest.raises(ValueError):
        opt.load_state_dict(sd)
    assert unchanged(opt, before)


def test_learning_rates_held_as_tensors_load_as_numbers():
    p, theirs = stepped(torch.optim.AdamW, 1)
    sd = copy.deepcopy(theirs.state_dict())
    sd["param_groups"][0]["lr"] = torch.tensor(0.25)
    _, opt = stepped(AdamW)
    opt.load_state_dict(sd)
    assert opt.param_groups[0]["lr"] == 0.25 and type(opt.param_groups[0]["lr"]) is float
    assert isinstance(sd["param_groups"][0]["lr"], torch.Tensor)  # the caller's dict stays as it was
