"""exp_avg for small beta1: a gradient beside a far larger average."""
import pytest
import torch

from ceo_firm_matching import AdamW

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("b1", [0.0, 1e-6, 0.3, 0.4999, 0.5, 0.9])
def test_average_after_a_large_gradient(device, bits, b1):
    if device != "cpu" and not torch.cuda.is_available():
        pytest.skip("no HIP device")
    lr, b2, n = 1e-2, 0.9, 1000
    gen = torch.Generator().manual_seed(3)
    p = torch.nn.Parameter(torch.zeros(n, device=device))
    opt = AdamW([p], lr=lr, betas=(b1, b2), eps=0.0, weight_decay=0.0, state_bits=bits)
    p.grad = (1e8 * (1 + torch.rand(n, generator=gen))).to(device)
    opt.step()
    m0, second = (x.reshape(-1)[:n].clone().cpu().double() for x in opt.held_states())
    v0 = second if bits == 32 else second.square()
    p0 = p.detach().cpu().double()
    g = 1 + torch.rand(n, generator=gen)
    p.grad = g.to(device)
    opt.step()
    gd, u = g.double(), 2.0 ** -24
    m = b1 * m0 + (1 - b1) * gd
    # one of m0 + (1 - b1)(g - m0) and g - b1 (g - m0), by the smaller factor: off by 4 u of |g| and of twice b1 |m0| (in
    # the first form b1 is at least 1/2)
    off = 4 * u * (gd.abs() + 2 * b1 * m0.abs())
    if bits == 32:
        got = opt.held_states()[0].reshape(-1)[:n].cpu().double()
        assert bool(((got - m).abs() <= off).all())
        if b1 == 0:
            assert torch.equal(got, gd)
    k, denom = lr / (1 - b1 ** 2), ((b2 * v0 + (1 - b2) * gd * gd) / (1 - b2 ** 2)).sqrt()
    want = p0 - k * m / denom
    tol = k * off / denom + 8 * u * k * m.abs() / denom + u * (p0.abs() + want.abs())
    assert bool(((p.detach().cpu().double() - want).abs() <= tol * 1.01).all())
