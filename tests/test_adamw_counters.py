"""tt_adamw_step with step counts on the device: a counter that several tensors
name, empty tensors, and what is refused."""
import ctypes

import numpy as np
import pytest
import torch

from ceo_firm_matching import AdamW, block8
from ceo_firm_matching import _native as N

HP = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


class Lists:
    """A list of tensors with its states and counters, stepped through the C-ABI."""

    def __init__(self, sizes, counter, n_counters, bits, dev, seed=5):
        g = torch.Generator().manual_seed(0)
        self.params = [torch.randn(n, generator=g).to(dev) for n in sizes]
        self.grads = [torch.randn(n, generator=g).to(dev) for n in sizes]
        self.bits, self.seed, self.dev = bits, seed, dev
        nb = [block8.blocks_of(n) for n in sizes]
        self.total = sum(nb)
        self.steps = torch.zeros(n_counters, dtype=torch.int64, device=dev)
        self.coefs = torch.zeros(n_counters, 4, device=dev)
        codes = lambda: torch.zeros(self.total, 128, dtype=torch.uint8, device=dev)  # noqa: E731
        scales = lambda: torch.full((self.total,), 127, dtype=torch.uint8, device=dev)  # noqa: E731
        self.arenas = ([torch.zeros(self.total, 128, device=dev) for _ in range(2)] if bits == 32 else
                       [codes(), scales(), codes(), scales()])
        names = ("exp_avg", "exp_avg_sq") if bits == 32 else ("m_codes", "m_scales", "r_codes", "r_scales")
        self.state = N.TTAdamWState(n_blocks=self.total, steps=self.steps.data_ptr(), coefs=self.coefs.data_ptr(), n_steps=n_counters,
                                    **{k: t.data_ptr() for k, t in zip(names, self.arenas)})
        self.list = (N.TTAdamWTensor * len(sizes))()
        at = 0
        for i, n in enumerate(sizes):
            self.list[i] = N.TTAdamWTensor(param=self.params[i].data_ptr() or None, grad=self.grads[i].data_ptr() or None, n=n,
                                           block0=at, step=counter[i], dtype=N.TT_F32)
            at += nb[i]

    def step(self):
        hp = N.TTAdamWHP(HP["lr"], *HP["betas"], HP["eps"], HP["weight_decay"])
        return N.lib().tt_adamw_step(self.list, len(self.list), self.bits, ctypes.byref(self.state), ctypes.byref(hp), self.seed,
                                     N.stream_ptr(self.dev) if self.dev.type == "cuda" else None)


@pytest.fixture
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    return torch.device("cuda:0")


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("counter", ["one", "few", "falling"])
def test_a_counter_that_tensors_share_advances_once_a_call(dev, bits, counter):
    """Three launches of tensors; the same values as with step counts on the host."""
    sizes = [37 * i % 300 + 1 for i in range(150)]
    at = {"one": [2] * 150, "few": [i % 5 for i in range(150)], "falling": [149 - i for i in range(150)]}[counter]
    n_counters = {"one": 4, "few": 5, "falling": 150}[counter]
    a = Lists(sizes, at, n_counters, bits, dev)
    want = [torch.nn.Parameter(p.clone()) for p in a.params]
    opt = AdamW(want, state_bits=bits, seed=a.seed, **HP)
    for t in range(1, 4):
        N.check(a.step(), "tt_adamw_step")
        for p, g in zip(want, a.grads):
            p.grad = g
        opt.step()
        steps = a.steps.tolist()
        assert [steps[k] for k in sorted(set(at))] == [t] * len(set(at)) and sum(steps) == t * len(set(at))
        for x, y in zip(a.params, want):
            assert torch.equal(x, y), t
        for x, y in zip(a.arenas, opt._buckets[0].arenas.values()):
            assert torch.equal(x, y), t


def test_refusals():
    cpu = torch.device("cpu")
    a = Lists([10, 20], [0, 1], 2, 32, cpu)
    for field, value in (("n_steps", 1), ("n_steps", 2 ** 32), ("coefs", None)):
        a = Lists([10, 20], [0, 1], 2, 32, cpu)
        setattr(a.state, field, value)
        assert a.step() == N.TT_ERR_ARG, field
    a = Lists([10, 20], [0, -1], 2, 32, cpu)
    assert a.step() == N.TT_ERR_ARG


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("shapes", [[(0, 4)], [(0, 4), (5,), (0,)], [(3,)] * 70 + [(0,)]])
def test_empty_parameters_count_their_steps(dev, bits, shapes):
    """As with step counts on the host."""
    counts = []
    for capturable in (False, True):
        params = [torch.nn.Parameter(torch.ones(s, device=dev)) for s in shapes]
        opt = AdamW(params, state_bits=bits, capturable=capturable)
        for _ in range(2):
            for p in params:
                p.grad = torch.ones_like(p)
            opt.step()
        counts.append([int(opt.state[p]["step"]) for p in params])
    assert counts[0] == counts[1] == [2] * len(shapes)


def test_the_counter_of_an_empty_tensor_is_checked():
    a = Lists([10, 0], [0, 7], 2, 32, torch.device("cpu"))
    assert a.step() == N.TT_ERR_ARG
