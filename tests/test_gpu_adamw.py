"""AdamW's HIP kernels (tt_adamw_*) against 64 bits and against the torch form
of the 8-bit states."""
import pytest
import torch

from ceo_firm_matching import AdamW
from ceo_firm_matching import block8

pytestmark = pytest.mark.gpu

HP = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


@pytest.fixture
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    return torch.device("cuda:0")


def make(shapes, dtypes, dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter((0.1 * torch.randn(s, generator=g)).to(dt).to(dev))
            for s, dt in zip(shapes, (dtypes * len(shapes))[:len(shapes)])]


def set_grads(params, seed):
    g = torch.Generator().manual_seed(seed)
    for p in params:
        p.grad = (1e-2 * torch.randn(p.shape, generator=g) * torch.exp(torch.randn((), generator=g))).to(p.dtype).to(p.device)


def check_step(opt, params, before, held, t, hp=HP):
    """One step from known states against 64 bits, the codes against the torch form."""
    a, b = (x.cpu() for x in opt.held_states())
    b1, b2 = hp["betas"]
    at, flips, total = 0, 0, 0
    for i, (p, p0) in enumerate(zip(params, before)):
        n, nb = p.numel(), block8.blocks_of(p.numel())
        get = lambda x: x[at:at + nb].reshape(-1)[:n].double()  # noqa: E731
        gd, pd = p.grad.cpu().reshape(-1).double(), p0.reshape(-1).double()
        m0 = get(held[0])
        v0 = get(held[1]) if opt._bits == 32 else get(held[1]).square()
        m = b1 * m0 + (1 - b1) * gd
        v = b2 * v0 + (1 - b2) * gd * gd
        denom = (v / (1 - b2 ** t)).sqrt() + hp["eps"]
        k = hp["lr"] / (1 - b1 ** t)
        pe = pd - hp["lr"] * hp["weight_decay"] * pd - k * m / denom
        # fp32, u = 2^-24: m' is off by at most 4 u (|m| + |g|), which the division by denom carries into p'; the
        # quotient, the step size, denom's roundings and the last product add 8 u of the update, decay's factor and
        # product 2 u |p|, the sum u |p'|; then one rounding to the parameter's type (fp16: half its smallest step)
        mags = m0.abs() + gd.abs()
        off = 2.0 ** -24 * (4 * k * mags / denom + 8 * k * m.abs() / denom + 2 * pd.abs() + pe.abs())
        tol = off * 1.01 + (pe.abs() + off) * torch.finfo(p.dtype).eps / 2 + (2.0 ** -25 if p.dtype == torch.float16 else 0)
        assert bool(((p.detach().cpu().reshape(-1).double() - pe).abs() <= tol).all()), (i, t)
        if opt._bits == 32:
            assert bool(((get(a) - m).abs() <= 4 * 2.0 ** -24 * mags).all()), (i, t)
            assert bool(((get(b) - v).abs() <= 6 * 2.0 ** -24 * v + 1e-44).all()), (i, t)
        elif n:
            pad = lambda x: torch.nn.functional.pad(x.float(), (0, -n % 128)).reshape(-1, 128)  # noqa: E731
            um, ur = block8.rounding_bits(opt._buckets[0].block0[i], nb, opt._seed, t)
            st = opt.state[p]
            for x, u, fmt, name, keep in ((m, um, block8.E4M3, "exp_avg", False), (v.sqrt(), ur, block8.E4M4, "exp_avg_sqrt", True)):
                codes, scales = block8.hold(pad(x), u, fmt, keep)
                assert torch.equal(st[name + "_scales"].cpu(), scales), (i, t, name)
                got, want = (c.reshape(-1)[:n].int() for c in (st[name + "_codes"].cpu(), codes))
                if fmt is block8.E4M3:  # by magnitude and sign: both codes of zero are zero
                    got, want = (torch.where(c >= 128, 128 - c, c) for c in (got, want))
                # the kernel's m and sqrt(v) are fp32: within 8 u of the border of two codes it may take the other
                assert int((got - want).abs().max()) <= 1
                flips += int((got != want).sum())
                total += n
                assert torch.equal(get(a if name == "exp_avg" else b), block8.held(
                    torch.nn.functional.pad(st[name + "_codes"].cpu().reshape(-1), (0, -n % 128)).reshape(-1, 128),
                    scales, fmt).reshape(-1)[:n].double())
        assert not a[at:at + nb].reshape(-1)[n:].any() and not b[at:at + nb].reshape(-1)[n:].any()
        at += nb
    # 8 u against a smallest step of 2^-4 of the value: 2^-17 of the places, and m's cancellations
    assert flips <= 3 + total * 2.0 ** -10, (flips, total)


SHAPES = {
    "one": [()],
    "edges": [(1,), (7,), (8,), (127,), (128,), (129,), (3, 43), (0, 4), (2047,), (2048,), (2049,), (16, 1000)],
    "list": [((37 * i) % 300 + 1,) for i in range(150)],  # more tensors than one launch takes
    "large": [(5, 100003), (1,)],
}


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("name", list(SHAPES))
def test_steps(dev, bits, name):
    params = make(SHAPES[name], [torch.float32, torch.bfloat16, torch.float16], dev)
    opt = AdamW(params, state_bits=bits, seed=11, **HP)
    for t in range(1, 4):
        held = [x.cpu().clone() for x in opt.held_states()]
        before = [p.detach().cpu().clone() for p in params]
        set_grads(params, 100 * t)
        opt.step()
        check_step(opt, params, before, held, t)


@pytest.mark.parametrize("bits", [32, 8])
def test_odd_addresses_and_gradient_layouts(dev, bits):
    """Parameters and gradients at any aligned address; gradients that are
    expanded or transposed."""
    store = [torch.zeros(4000, device=dev), torch.zeros(4000, dtype=torch.bfloat16, device=dev)]
    params = [torch.nn.Parameter(store[0][3:1003].view(10, 100)), torch.nn.Parameter(store[1][1:778].view(7, 111)),
              torch.nn.Parameter(store[1][1001:1131])]
    opt = AdamW(params, state_bits=bits, **HP)
    with torch.no_grad():
        for p in params:
            p.copy_(torch.randn(p.shape))
    for t in range(1, 3):
        held = [x.cpu().clone() for x in opt.held_states()]
        before = [p.detach().cpu().clone() for p in params]
        params[0].grad = torch.randn(100, 10, device=dev).t()
        params[1].grad = torch.zeros(900, dtype=torch.bfloat16, device=dev)[5:782].view(7, 111) + 0.25
        params[2].grad = torch.full((1,), 0.5, dtype=torch.bfloat16, device=dev).expand(130)
        opt.step()
        check_step(opt, params, before, held, t)
    untouched = torch.ones(4000, dtype=torch.bool)
    untouched[3:1003] = False
    assert not store[0].cpu()[untouched].any()
    untouched[:] = True
    untouched[1:778] = untouched[1001:1131] = False
    assert not store[1].cpu()[untouched].any()


@pytest.mark.parametrize("bits", [32, 8])
def test_repeatable_and_equal_to_the_cpu_form(dev, bits):
    runs = []
    for device in (dev, dev, torch.device("cpu")):
        params = make([(300, 17), (5,)], [torch.float32], device, 3)
        opt = AdamW(params, state_bits=bits, seed=2, **HP)
        for t in range(4):
            set_grads(params, t)
            opt.step()
        runs.append(torch.cat([p.detach().cpu().reshape(-1) for p in params]))
    assert torch.equal(runs[0], runs[1])
    # 8 bits: a code that fell on the other side moves one update by at most its step of 2^-3
    d = (runs[0] - runs[2]).abs()
    if bits == 32:
        assert float(d.max()) <= 4 * 16 * 2.0 ** -24 * (0.5 + 4 * HP["lr"] * 12)
    else:
        assert float((d > 1e-6).float().mean()) <= 2.0 ** -8 and float(d.max()) <= 4 * HP["lr"]


@pytest.mark.parametrize("bits", [32, 8])
def test_nonfinite_and_missing_gradients(dev, bits):
    p, q = make([(500,), (40,)], [torch.float32], dev)
    opt = AdamW([p, q], state_bits=bits, **HP)
    q0 = q.detach().clone()
    g = torch.full((500,), 0.5, device=dev)
    g[7], g[300], g[301] = float("nan"), float("inf"), -float("inf")
    bad = ~torch.isfinite(g)
    p.grad = g
    for _ in range(3):
        opt.step()
    assert torch.equal(torch.isnan(p.detach()), bad)
    assert torch.equal(q.detach(), q0) and int(opt.state[q]["step"]) == 0 and int(opt.state[p]["step"]) == 3
    for _ in range(2):  # different step counts in one launch
        q.grad = torch.full((40,), 0.5, device=dev)
        opt.step()
    want = AdamW([q2 := torch.nn.Parameter(q0.clone())], state_bits=bits, **HP)
    for _ in range(2):
        q2.grad = torch.full((40,), 0.5, device=dev)
        want.step()
    if bits == 32:  # (8 bits: the rounding hash goes by the place in the arena)
        assert torch.equal(q.detach(), q2.detach())
    assert int(opt.state[p]["step"]) == 5


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_equal_eager_ones(dev, bits):
    """capturable: device step counts; replays with eager work between them."""
    shapes = [((53 * i) % 400 + 1,) for i in range(70)]  # two launches
    a, b = make(shapes, [torch.float32, torch.bfloat16], dev), make(shapes, [torch.float32, torch.bfloat16], dev)
    oa = AdamW(a, state_bits=bits, seed=5, **HP)
    ob = AdamW(b, state_bits=bits, seed=5, capturable=True, **HP)
    set_grads(a, 1)
    set_grads(b, 1)
    static = [p.grad for p in b]
    oa.step()
    ob.step()
    with pytest.raises(RuntimeError, match="capturable"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            oa.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ob.step()
    for k in range(4):
        set_grads(a, 10 + k)
        for s, p in zip(static, a):
            s.copy_(p.grad)
        oa.step()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(a, b):
            assert torch.equal(x, y), k
        for x, y in zip(oa.held_states(), ob.held_states()):
            assert torch.equal(x, y), k
    assert int(ob.state[b[0]]["step"]) == 5
    set_grads(a, 99)
    set_grads(b, 99)
    oa.step()
    ob.step()  # eager again after the replays
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_another_stream(dev):
    a, b = make([(100000,)], [torch.float32], dev), make([(100000,)], [torch.float32], dev)
    oa, ob = AdamW(a, **HP), AdamW(b, **HP)
    s = torch.cuda.Stream()
    for t in range(3):
        set_grads(a, t)
        set_grads(b, t)
        oa.step()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            ob.step()
        torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(a[0], b[0])


def test_long_run_tracks_the_second_moment(dev):
    """Under gradients of constant size the 8-bit root settles where the
    32-bit one does: rounding to nearest would freeze it on the way.  The root
    of each value carries the noise of the roundings: per step a jump of one
    code, 1/16 of it at most, as often as the drift calls for; summed over the
    1 / (1 - b2) steps of memory 2^-4 sqrt(1/2) sqrt(0.05/2) stays below 1 %
    of the mean over 10,000 values; 5 % is asked."""
    p8, p32 = (torch.nn.Parameter(torch.zeros(10000, device=dev)) for _ in range(2))
    o8, o32 = AdamW([p8], state_bits=8, betas=(0.9, 0.99)), AdamW([p32], betas=(0.9, 0.99))
    g = torch.Generator(device=dev).manual_seed(1)
    for _ in range(500):
        p8.grad = p32.grad = torch.randn(10000, generator=g, device=dev)
        o8.step()
        o32.step()
    m8, r8 = (x.float().reshape(-1)[:10000] for x in o8.held_states())
    m32, v32 = (x.reshape(-1)[:10000] for x in o32.held_states())
    assert abs(float(r8.square().mean() / v32.mean()) - 1) < 0.05
    assert abs(float((m8 * m32).mean() / m32.square().mean()) - 1) < 0.05


@pytest.mark.parametrize("bits", [32, 8])
def test_more_than_2_31_values(dev, bits):
    n = 2 ** 31 + 1000
    p = torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16, device=dev))
    opt = AdamW([p], lr=1e-2, state_bits=bits, weight_decay=0.0)
    g = torch.zeros(n, dtype=torch.bfloat16, device=dev)
    places = [0, 2 ** 31 - 1, 2 ** 31, n - 1]
    for at in places:
        g[at] = 1.0
    p.grad = g
    opt.step()
    assert sum(int(part.count_nonzero()) for part in p.detach().split(1 << 28)) == 4
    # the first step moves by lr whatever the gradient's size
    assert [float(p.detach()[at]) for at in places] == [float(torch.tensor(-1e-2).bfloat16())] * 4


def test_a_refused_step_changes_nothing(dev):
    (p,) = make([(50,)], [torch.float32], dev)
    opt = AdamW([p])
    p.grad = torch.ones(50, device=dev)
    before = p.detach().clone()
    opt.param_groups[0]["lr"] = float("nan")
    with pytest.raises(ValueError):
        opt.step()
    assert torch.equal(p.detach(), before) and int(opt.state[p]["step"]) == 0
    opt.param_groups[0]["lr"] = 1e-3
    opt.step()
    assert int(opt.state[p]["step"]) == 1 and not torch.equal(p.detach(), before)
