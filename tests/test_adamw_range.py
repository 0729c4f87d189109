"""AdamW over the whole range of float32: second moments that are subnormal,
with eps = 0 too."""
import pytest
import torch

from ceo_firm_matching import AdamW

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [0.0, 1e-21])
def test_subnormal_second_moments(device, bits, eps):
    if device != "cpu" and not torch.cuda.is_available():
        pytest.skip("no HIP device")
    lr, b1, b2, n = 1e-2, 0.9, 0.99, 5000
    gen = torch.Generator().manual_seed(1)
    want_v = torch.exp2(-145 + 30 * torch.rand(n, generator=gen, dtype=torch.float64))  # both sides of 2^-126
    g = ((want_v / (1 - b2)).sqrt() * torch.where(torch.rand(n, generator=gen) < 0.5, -1.0, 1.0)).float()
    p = torch.nn.Parameter(torch.zeros(n, device=device))
    opt = AdamW([p], lr=lr, betas=(b1, b2), eps=eps, weight_decay=0.0, state_bits=bits)
    p.grad = g.to(device)
    opt.step()
    gd = g.double()
    v = (1 - b2) * gd * gd
    move = lr * gd / (gd.abs() + eps)  # the first step's bias corrections cancel
    # v' is a product rounded to float32's grid, 2^-149 apart below 2^-126: off by 2^-150 there, half of that relative
    # to the root; 24 u for the rest of the arithmetic (u = 2^-24)
    off = (p.detach().cpu().double() + move).abs()
    tol = move.abs() * (0.55 * 2.0 ** -150 / v + 24 * 2.0 ** -24)
    assert bool((off <= tol).all()), float((off / tol).max())
    held = opt.held_states()[1].cpu().reshape(-1)[:n]
    assert bool((held > 0).all())  # a positive root (or square) is never held as zero
    # ... so that the next step, with no gradient at all, moves by a finite amount
    p.grad = torch.zeros(n, device=device)
    opt.step()
    assert bool(torch.isfinite(p.detach()).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [32, 8])
def test_zero_gradients_beside_tiny_ones(device, bits):
    if device != "cpu" and not torch.cuda.is_available():
        pytest.skip("no HIP device")
    p = torch.nn.Parameter(torch.ones(1000, device=device))
    opt = AdamW([p], lr=1e-2, eps=1e-30, weight_decay=0.0, state_bits=bits)
    g = torch.zeros(1000, device=device)
    g[::7] = 3e-21
    p.grad = g
    opt.step()
    # v' = 9e-45 is 6.4 steps of 2^-149, held as 6: the root is 3.3 % low
    moved = (1 - p.detach()).cpu()
    assert bool((moved[g.cpu() == 0] == 0).all())
    assert bool(((moved[::7] / 1e-2 - 1).abs() < 0.1).all())
