"""AdamW over many tensors, on the CPU: the formulas against 64 bits, the 8-bit
states' codes, state_dict, and what is refused (also by the C-ABI)."""
import copy
import ctypes

import numpy as np
import pytest
import torch

from ceo_firm_matching import AdamW
from ceo_firm_matching import _native as N
from ceo_firm_matching import block8


def exact_step(p, g, m, v, t, lr, b1, b2, eps, wd):
    """One step in 64 bits."""
    p, g, m, v = (x.double() for x in (p, g, m, v))
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    p = p - lr * wd * p - lr * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + eps)
    return p, m, v


def grid_step(y, mant, scale):
    """Distance of neighbouring codes at magnitude y under a block scale."""
    return torch.exp2(torch.floor(torch.log2((y / scale).clamp_min(2.0 ** -6))) - mant) * scale


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_steps_follow_the_formula(bits, dtype):
    torch.manual_seed(1)
    params = [torch.nn.Parameter((0.1 * torch.randn(s)).to(dtype)) for s in ((3, 50), (128,), (), (1, 257), (0, 4))]
    hp = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
    opt = AdamW(params, state_bits=bits, seed=3, **hp)
    for t in range(1, 5):
        held = [x.clone() for x in opt.held_states()]
        before = [p.detach().clone() for p in params]
        for p in params:
            p.grad = (1e-2 * torch.randn(p.shape)).to(dtype)
        opt.step()
        a, b = opt.held_states()
        at = 0
        for p, p0 in zip(params, before):
            n, nb = p.numel(), block8.blocks_of(p.numel())
            get = lambda x: x[at:at + nb].reshape(-1)[:n].double()  # noqa: E731
            m0, v0 = get(held[0]), get(held[1]) if bits == 32 else get(held[1]).square()
            pe, me, ve = exact_step(p0.reshape(-1), p.grad.reshape(-1), m0, v0, t, *(hp["lr"], *hp["betas"], hp["eps"], 0.1))
            # fp32, u = 2^-24: m' = m + w (g - m) is off by at most 4 u (|m| + |g|) (its parts may cancel), which the
            # division by denom carries into p'; the quotient, the step size, denom's five roundings and the last
            # product add 8 u of the update, decay's factor and product 2 u |p|, the sum u |p'|; then one rounding
            # to the parameter's type
            gd, pd = p.grad.reshape(-1).double(), p0.reshape(-1).double()
            mags = m0.abs() + gd.abs()
            denom = (ve / (1 - hp["betas"][1] ** t)).sqrt() + hp["eps"]
            k = hp["lr"] / (1 - hp["betas"][0] ** t)
            off = 2.0 ** -24 * (4 * k * mags / denom + 8 * k * me.abs() / denom + 2 * pd.abs() + pe.abs())
            tol = off * 1.01 + (pe.abs() + off) * torch.finfo(dtype).eps / 2
            if dtype == torch.float16:
                tol = tol + 2.0 ** -25
            assert bool(((p.detach().reshape(-1).double() - pe).abs() <= tol).all())
            if bits == 32:
                assert bool(((get(a) - me).abs() <= 4 * 2.0 ** -24 * mags).all())
                assert bool(((get(b) - ve).abs() <= 6 * 2.0 ** -24 * ve).all())
            elif n:
                for got, want, codes, mant in ((get(a), me, opt.state[p]["exp_avg_scales"], 3),
                                               (get(b), ve.sqrt(), opt.state[p]["exp_avg_sqrt_scales"], 4)):
                    s = torch.exp2(codes.double() - 127).repeat_interleave(128)[:n]
                    assert bool(((got - want).abs() <= grid_step(want.abs(), mant, s) * (1 + 1e-5)).all())
                assert bool((get(b)[ve > 0] > 0).all())
            pad = a[at:at + nb].reshape(-1)[n:], b[at:at + nb].reshape(-1)[n:]
            assert all(not x.any() for x in pad)
            at += nb


def test_codes_are_a_grid_and_rounding_is_unbiased():
    """Every code decodes to its e4m3 / e4m4 value and encodes to itself; the
    mean over many roundings of one value is the value."""
    for fmt, top in ((block8.E4M3, 0x7E), (block8.E4M4, 0xFE)):
        mant = fmt[0]
        codes = torch.zeros(2, 128, dtype=torch.uint8)
        codes.reshape(-1)[:top + 1] = torch.arange(top + 1).to(torch.uint8)
        codes[:, 127] = top  # the largest code in each block fixes its scale
        v = block8.held(codes, torch.tensor([127, 127]), fmt)
        c = codes.double()
        e, f = torch.floor(c / 2 ** mant), c % 2 ** mant
        want = torch.where(e > 0, (1 + f / 2 ** mant) * 2.0 ** (e - 7), f / 2 ** mant * 2.0 ** -6)
        assert torch.equal(v.double(), want)
        got, s = block8.hold(v, torch.zeros(2, 128, dtype=torch.int64), fmt, False)
        assert torch.equal(got, codes) and s.tolist() == [127, 127]
    x = torch.full((2000, 128), 1.03)
    x[:, 0] = 400.0
    um, ur = block8.rounding_bits(0, 2000, 5, 9)
    for u, fmt, rel in ((um, block8.E4M3, 1 / 8), (ur, block8.E4M4, 1 / 16)):
        v = block8.held(*block8.hold(x, u, fmt, False), fmt)[:, 1:].double()
        # 254,000 draws of a step of `rel`: the mean is within 5 standard errors
        assert abs(float(v.mean()) - float(x[0, 1])) < 5 * rel / 2 / (2000 * 127) ** 0.5
        assert v.unique().numel() == 2


def test_nonfinite_gradients_stay_where_they_are():
    for bits in (32, 8):
        p = torch.nn.Parameter(torch.ones(300))
        opt = AdamW([p], lr=0.1, state_bits=bits)
        g = torch.full((300,), 0.5)
        g[7], g[130] = float("nan"), float("inf")
        p.grad = g
        opt.step()
        opt.step()
        bad = torch.zeros(300, dtype=torch.bool)
        bad[7] = bad[130] = True
        assert torch.equal(torch.isnan(p.detach()), bad), bits
        assert torch.isfinite(p.detach()[~bad]).all()


def test_zero_gradients_keep_zero_states_and_skipped_parameters_stand_still():
    for bits in (32, 8):
        p, q = torch.nn.Parameter(torch.ones(200)), torch.nn.Parameter(torch.ones(5))
        opt = AdamW([p, q], lr=0.1, weight_decay=0.0, state_bits=bits)
        p.grad = torch.zeros(200)
        for _ in range(3):
            opt.step()
        assert torch.equal(p.detach(), torch.ones(200)) and torch.equal(q.detach(), torch.ones(5))
        assert all(not x.any() for x in opt.held_states())
        assert int(opt.state[p]["step"]) == 3 and int(opt.state[q]["step"]) == 0


def _run(opt, params, steps, seed):
    g = torch.Generator().manual_seed(seed)
    for _ in range(steps):
        for p in params:
            p.grad = torch.randn(p.shape, generator=g).to(p.device, p.dtype)
        opt.step()


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_round_trip_and_copies(bits):
    torch.manual_seed(0)
    mk = lambda: [torch.nn.Parameter(torch.linspace(-1, 1, n).to(dt)) for n, dt in ((130, torch.float32), (7, torch.bfloat16))]  # noqa: E731
    a, b = mk(), mk()
    oa, ob = AdamW(a, lr=0.01, state_bits=bits, seed=4), AdamW(b, lr=0.5, state_bits=bits, seed=4)
    _run(oa, a, 3, 1)
    sd = copy.deepcopy(oa.state_dict())
    arenas = [x.data_ptr() for x in ob._buckets[0].arenas.values()]
    ob.load_state_dict(sd)
    assert [x.data_ptr() for x in ob._buckets[0].arenas.values()] == arenas  # captured steps keep their memory
    with torch.no_grad():
        for x, y in zip(a, b):
            y.copy_(x)
    oc = copy.deepcopy(ob)
    c = oc.param_groups[0]["params"]
    _run(oa, a, 2, 2)
    _run(ob, b, 2, 2)
    _run(oc, c, 2, 2)
    for x, y, z in zip(a, b, c):
        assert torch.equal(x, y) and torch.equal(x, z)
    assert ob.param_groups[0]["lr"] == 0.01 and int(ob.state[b[0]]["step"]) == 5


def test_loads_torch_adamw_states_and_follows_it():
    torch.manual_seed(0)
    a = [torch.nn.Parameter(torch.randn(40, 3)), torch.nn.Parameter(torch.randn(7))]
    b = [torch.nn.Parameter(x.detach().clone()) for x in a]
    oa, ob = torch.optim.AdamW(a, lr=1e-2), AdamW(b, lr=1e-2)
    _run(oa, a, 2, 1)
    ob.load_state_dict(oa.state_dict())
    with torch.no_grad():
        for x, y in zip(a, b):
            y.copy_(x)
    _run(oa, a, 3, 2)
    _run(ob, b, 3, 2)
    for x, y in zip(a, b):
        # three steps of at most lr(1 + wd): each side rounds values <= 4 a few times
        assert float((x - y).detach().abs().max()) <= 3 * 8 * 2.0 ** -24 * 4


def test_groups_schedulers_and_closures():
    p, q = torch.nn.Parameter(torch.ones(3)), torch.nn.Parameter(torch.ones(3))
    opt = AdamW([{"params": [p]}, {"params": [q], "lr": 0.0, "weight_decay": 0.0}], lr=0.1)
    sched = torch.optim.lr_scheduler.StepLR(opt, 1, 0.5)

    def closure():
        opt.zero_grad()
        loss = (p.sum() + q.sum()) * 2
        loss.backward()
        return loss

    assert float(opt.step(closure)) == 12.0
    sched.step()
    assert torch.equal(q.detach(), torch.ones(3)) and float(p[0]) < 1 and opt.param_groups[0]["lr"] == 0.05
    opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(2))]})
    assert len(opt._buckets) == 3


def test_refusals():
    p = torch.nn.Parameter(torch.ones(4))
    for kw in (dict(state_bits=16), dict(lr=-1.0), dict(lr=float("nan")), dict(betas=(1.0, 0.9)), dict(eps=-1e-8),
               dict(weight_decay=-0.1), dict(capturable=True)):
        with pytest.raises(ValueError):
            AdamW([p], **kw)
    with pytest.raises(NotImplementedError):
        AdamW([torch.nn.Parameter(torch.ones(4, dtype=torch.float64))])
    with pytest.raises(ValueError):
        AdamW([torch.nn.Parameter(torch.ones(4, 3).t())])
    both = torch.zeros(10)
    with pytest.raises(ValueError, match="share memory"):
        AdamW([torch.nn.Parameter(both[:6]), torch.nn.Parameter(both[5:])])
    AdamW([torch.nn.Parameter(both[:5]), torch.nn.Parameter(both[5:])])
    opt = AdamW([p], state_bits=8)
    with pytest.raises(ValueError):
        opt.load_state_dict(AdamW([p]).state_dict())  # 32-bit states into 8-bit ones
    with pytest.raises(ValueError):
        opt.load_state_dict(AdamW([p, torch.nn.Parameter(torch.ones(1))], state_bits=8).state_dict())
    e = torch.nn.Embedding(4, 2, sparse=True)
    o = AdamW(e.parameters())
    e(torch.tensor([1])).sum().backward()
    with pytest.raises(NotImplementedError):
        o.step()
    p.grad = torch.ones(4)
    for other in (torch.ones(9), torch.ones(4, dtype=torch.bfloat16), torch.ones(8)[::2]):
        q = torch.nn.Parameter(torch.ones(4))
        o = AdamW([q], state_bits=8)
        q.data = other
        q.grad = torch.ones_like(other)
        with pytest.raises(RuntimeError, match="parameter changed"):
            o.step()
    q = torch.nn.Parameter(torch.ones(9))
    q.grad = torch.ones(9)
    q.data = torch.ones(4)  # the gradient is of the old size
    o = AdamW([q])
    with pytest.raises(RuntimeError, match="gradient"):
        o.step()


def test_host_argument_errors():
    """tt_adamw_*: decided on the host before anything is enqueued."""
    L = N.lib()
    buf = np.zeros(1 << 16, dtype=np.float32)
    at = buf.ctypes.data
    st = N.TTAdamWState(exp_avg=at, exp_avg_sq=at, m_codes=at, m_scales=at, r_codes=at, r_scales=at, n_blocks=4)
    hp = N.TTAdamWHP(1e-3, 0.9, 0.999, 1e-8, 0.01)

    def call(bits=32, state=st, h=hp, n_t=1, **kw):
        t = N.TTAdamWTensor(param=at, grad=at, n=300, block0=0, step=1, dtype=N.TT_F32)
        for k, v in kw.items():
            setattr(t, k, v)
        return L.tt_adamw_step(ctypes.byref(t), n_t, bits, state and ctypes.byref(state), h and ctypes.byref(h), 0, None)

    assert call(n=0) == N.TT_OK and call(n_t=0) == N.TT_OK
    assert call(bits=16) == N.TT_ERR_UNSUPPORTED
    for kw in (dict(param=None), dict(grad=None), dict(n=-1), dict(step=0), dict(dtype=3), dict(block0=2), dict(block0=-1),
               dict(n=513), dict(param=at + 2), dict(n_t=-1), dict(state=None), dict(h=None),
               dict(h=N.TTAdamWHP(1e-3, 1.0, 0.999, 1e-8, 0.01)), dict(h=N.TTAdamWHP(float("nan"), 0.9, 0.999, 1e-8, 0.01)),
               dict(state=N.TTAdamWState(n_blocks=4)), dict(bits=8, state=N.TTAdamWState(exp_avg=at, exp_avg_sq=at, n_blocks=4)),
               dict(state=N.TTAdamWState(exp_avg=at, exp_avg_sq=at, n_blocks=4, steps=at)),
               dict(state=N.TTAdamWState(exp_avg=at, exp_avg_sq=at, n_blocks=4, steps=at, coefs=at, n_steps=1)),
               dict(block0=2 ** 62), dict(n=2 ** 62), dict(grad=at + 1, dtype=N.TT_BF16),
               dict(state=N.TTAdamWState(exp_avg=at + 2, exp_avg_sq=at, n_blocks=4))):
        assert call(**kw) == N.TT_ERR_ARG, kw
    assert L.tt_adamw_held(None, at, at, None) == N.TT_ERR_ARG
    assert L.tt_adamw_held(ctypes.byref(st), None, at, None) == N.TT_ERR_ARG
    for which, s in ((N.TT_STRUCT_ADAMW_TENSOR, N.TTAdamWTensor), (N.TT_STRUCT_ADAMW_STATE, N.TTAdamWState),
                     (N.TT_STRUCT_ADAMW_HP, N.TTAdamWHP)):
        assert L.tt_struct_size(which) == ctypes.sizeof(s)
