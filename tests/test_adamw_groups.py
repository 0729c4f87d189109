"""A step over several parameter groups is taken whole or not at all."""
import pytest
import torch

from ceo_firm_matching import AdamW

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]


def make(device, bits):
    if device != "cpu" and not torch.cuda.is_available():
        pytest.skip("no HIP device")
    params = [torch.nn.Parameter(torch.ones(n, device=device)) for n in (300, 20, 5)]
    opt = AdamW([{"params": [p]} for p in params], lr=1e-2, state_bits=bits)
    for p in params:
        p.grad = torch.full_like(p, 0.5)
    opt.step()
    return params, opt


def everything(params, opt):
    return ([p.detach().clone() for p in params] + [x.clone() for k in range(3) for x in opt.held_states(k)]
            + [opt.state[p]["step"].clone() for p in params])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [32, 8])
def test_a_refusal_in_a_later_group_leaves_the_earlier_ones(device, bits):
    params, opt = make(device, bits)

    def refused(error):
        before = everything(params, opt)
        with pytest.raises(error):
            opt.step()
        assert all(torch.equal(a, b) for a, b in zip(everything(params, opt), before))

    for key, value in (("lr", -1.0), ("eps", float("nan")), ("betas", (0.9, 1.5)), ("weight_decay", float("inf"))):
        good = opt.param_groups[2][key]
        opt.param_groups[2][key] = value
        refused(ValueError)
        opt.param_groups[2][key] = good
    last = params[2]
    last.grad = torch.sparse_coo_tensor(torch.tensor([[1]]), torch.tensor([1.0]), (5,)).to(device)
    refused(NotImplementedError)
    last.grad = None
    old = last.data
    last.data = torch.ones(7, device=device)
    last.grad = torch.ones(7, device=device)
    refused(RuntimeError)
    last.data, last.grad = old, torch.full_like(old, 0.5)
    opt.step()
    assert [int(opt.state[p]["step"]) for p in params] == [2, 2, 2]


@pytest.mark.gpu
def test_a_capture_is_refused_before_any_group_steps():
    params, opt = make("cuda:0", 32)
    host = torch.nn.Parameter(torch.ones(4))
    both = AdamW([{"params": [host]}, {"params": [params[0]]}], lr=1e-2)
    host.grad = torch.ones(4)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="capturable"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            both.step()
    torch.cuda.synchronize()
    assert torch.equal(host.detach(), torch.ones(4)) and int(both.state[host]["step"]) == 0
