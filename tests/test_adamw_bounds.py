"""The bounds of AdamW's hyperparameters: the same on CPU, on a HIP device and
behind the C-ABI."""
import ctypes

import numpy as np
import pytest
import torch

from ceo_firm_matching import AdamW
from ceo_firm_matching import _native as N

BAD = [("lr", -1e-3), ("lr", float("inf")), ("lr", float("nan")), ("weight_decay", -0.1), ("weight_decay", float("inf")),
       ("eps", -1e-8), ("eps", float("inf")), ("eps", float("nan")), ("betas", (-0.1, 0.9)), ("betas", (0.9, 1.0)),
       ("betas", (float("nan"), 0.9))]


@pytest.mark.parametrize("key,value", BAD)
def test_c_abi(key, value):
    buf = np.zeros(1024, dtype=np.float32)
    at = buf.ctypes.data
    st = N.TTAdamWState(exp_avg=at, exp_avg_sq=at, m_codes=at, m_scales=at, r_codes=at, r_scales=at, n_blocks=4)
    t = N.TTAdamWTensor(param=at, grad=at, n=300, block0=0, step=1, dtype=N.TT_F32)
    hp = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
    hp[key] = value
    h = N.TTAdamWHP(hp["lr"], *hp["betas"], hp["eps"], hp["weight_decay"])
    for bits in (8, 32):
        assert N.lib().tt_adamw_step(ctypes.byref(t), 1, bits, ctypes.byref(st), ctypes.byref(h), 0, None) == N.TT_ERR_ARG
    assert not buf.any()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("key,value", BAD)
def test_set_between_steps(device, key, value):
    """As a schedule may: the step raises and changes nothing."""
    if device != "cpu" and not torch.cuda.is_available():
        pytest.skip("no HIP device")
    p = torch.nn.Parameter(torch.ones(200, device=device))
    opt = AdamW([p], lr=1e-2)
    p.grad = torch.full((200,), 0.5, device=device)
    opt.step()
    before, m = p.detach().clone(), opt.held_states()[0].clone()
    good = opt.param_groups[0][key]
    opt.param_groups[0][key] = value
    with pytest.raises(ValueError):
        opt.step()
    assert torch.equal(p.detach(), before) and torch.equal(opt.held_states()[0], m) and int(opt.state[p]["step"]) == 1
    opt.param_groups[0][key] = good
    opt.step()
    assert int(opt.state[p]["step"]) == 2
