"""The embedding catalogue's HIP kernels (tt_cat_*) against the torch form and
against 64 bits."""
import pytest
import torch

from ceo_firm_matching import EmbeddingCatalogue
from ceo_firm_matching import block8

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    return torch.device("cuda:0")


def rows_of(m, d, seed, dtype=torch.float32, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(m, d, generator=g) * torch.exp(spread * torch.randn(m, 1, generator=g))).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,d", [(1, 1), (3, 60), (17, 128), (5, 129), (33, 250), (9, 513), (700, 64)])
def test_write_and_read_equal_the_torch_form(dev, m, d, dtype):
    x = rows_of(m, d, m + d, dtype, 1.0 if dtype == torch.float16 else 3.0)
    cat = EmbeddingCatalogue(m + 7, d, device=dev)
    cat.write(x.to(dev), start=4)
    codes, scales = block8.encode(x)
    assert torch.equal(cat.codes[4:4 + m].cpu(), codes) and torch.equal(cat.scales[4:4 + m].cpu(), scales)
    assert not cat.codes[:4].any() and not cat.codes[4 + m:].any()
    assert (cat.scales[:4] == 127).all() and (cat.scales[4 + m:] == 127).all()
    want = block8.decode(cat.codes.cpu(), cat.scales.cpu(), d)
    assert torch.equal(cat.read().cpu(), want)
    for dt in (torch.bfloat16, torch.float16):
        assert torch.equal(cat.read(dtype=dt).cpu(), want.to(dt))
    rows = torch.tensor([m + 6, -1, 4, m + 7, 4, 2 ** 40, -2 ** 40])
    got = cat.read(rows=rows.to(dev)).cpu()
    assert torch.equal(got[0], want[m + 6]) and torch.equal(got[2], want[4]) and torch.equal(got[4], want[4])
    assert not got[1].any() and not got[3].any() and not got[5:].any()


def test_every_value_scale_and_edge(dev):
    """All codes at all scales; the border of a scale; halfway values; tiny,
    huge, infinite and NaN values."""
    v = torch.arange(256).to(torch.uint8).view(torch.float8_e4m3fn).float()
    v = v[torch.isfinite(v)]
    v = torch.cat([v, torch.full((256 - v.numel(),), 448.0)]).reshape(2, 128)
    v[0, 0] = 448.0
    mid = (v + torch.roll(v, 1, 1)) / 2  # ties among them
    x = torch.cat([w * 2.0 ** e for e in range(-100, 120, 3) for w in (v, mid)])
    g = torch.Generator().manual_seed(0)
    bits = torch.randint(-2 ** 31, 2 ** 31, (400, 128), generator=g).to(torch.int32).view(torch.float32)  # any floats
    edge = torch.zeros(4, 128)
    edge[0, :3] = torch.tensor([float("inf"), -float("inf"), 2.0])
    edge[1, 5], edge[2, 0], edge[3, 1] = 1e-45, 3e38, 448.00003
    x = torch.cat([x, bits, edge])
    cat = EmbeddingCatalogue(x.shape[0], 128, device=dev)
    cat.write(x.to(dev))
    codes, scales = block8.encode(x)
    assert torch.equal(cat.scales.cpu(), scales)
    got = cat.codes.cpu()
    nan = (codes & 0x7F) == 0x7F
    assert torch.equal((got & 0x7F) == 0x7F, nan) and torch.equal(got[~nan], codes[~nan])
    r, want = cat.read().cpu(), block8.decode(codes, scales, 128)
    assert torch.equal(torch.isnan(r), torch.isnan(want)) and torch.equal(r[~nan], want[~nan])


@pytest.mark.parametrize("m", [3, 1000, 70001])
def test_indexed_writes(dev, m):
    """Rows named twice take their last mention, strays are left out, every
    other row stays as it was; twice in a row, and from int32 numbers."""
    d, cap = 40, 5000
    g = torch.Generator().manual_seed(m)
    cat, ref = EmbeddingCatalogue(cap, d, device=dev), EmbeddingCatalogue(cap, d)
    for k, dt in enumerate((torch.int64, torch.int32, torch.int64)):
        x = torch.randn(m, d, generator=g)
        rows = torch.randint(-50, cap + 50, (m,), generator=g).to(dt)
        cat.write(x.to(dev), rows=rows.to(dev))
        ref.write(x, rows=rows)
        assert torch.equal(cat.codes.cpu(), ref.codes) and torch.equal(cat.scales.cpu(), ref.scales), k
        assert not cat._owner.any()


def test_strided_rows(dev):
    x = rows_of(50, 300, 1).to(dev)
    for view in (x[:, 3:103], x[::2, :100], x.t()[:100, :40], x[:, ::3], x[:1, :100].expand(50, 100)):
        cat = EmbeddingCatalogue(view.shape[0], view.shape[1], device=dev)
        cat.write(view)
        codes, scales = block8.encode(view.cpu())
        assert torch.equal(cat.codes.cpu(), codes) and torch.equal(cat.scales.cpu(), scales)


def score_case(dev, m, n, d, dtype, out_dtype, seed=0):
    c = torch.nn.functional.normalize(rows_of(n, d, seed + 1), dim=1)
    q = torch.nn.functional.normalize(rows_of(m, d, seed + 2), dim=1).to(dtype)
    cat = EmbeddingCatalogue(n, d, device=dev)
    cat.write(c.to(dev))
    return cat, q.to(dev).requires_grad_(), torch.randn(m, n, generator=torch.Generator().manual_seed(seed)).to(out_dtype)


def check_scores(cat, q, s, n=None):
    n = cat.capacity if n is None else n
    d = cat.dim
    cv = cat.read()[:n].cpu().double()
    qv = block8.decode(*block8.encode(q.detach().cpu()), d).double()
    want, mags = qv @ cv.t(), qv.abs() @ cv.abs().t()
    # one rounding to the result's type (fp16: half its smallest step), and
    # 32 bits: products are exact, each of the at most d + 2 sums (truncated ones allowed for) is off by 2^-23
    # 16 bits: the 8-bit matrix instruction cuts products off below the largest of a block's, 128 of them by 2^-18 of
    # it at most: 2^-11, once more for the sum over the blocks
    tol = torch.finfo(s.dtype).eps / 2 * want.abs() * 1.01 + (d + 2) * 2.0 ** -23 * mags
    if s.dtype != torch.float32:
        big = lambda x: torch.nn.functional.pad(x.abs(), (0, -d % 128)).reshape(x.shape[0], -1, 128).amax(2)  # noqa: E731
        tol = tol + 2.0 ** -10 * (big(qv) @ big(cv).t())
    tol = tol + (2.0 ** -25 if s.dtype == torch.float16 else 0.0)
    off = (s.detach().cpu().double() - want).abs()
    assert bool((off <= tol).all()), float((off / tol).max())


def check_dq(cat, q, ds, dq, n=None):
    n = cat.capacity if n is None else n
    cv = cat.read()[:n].cpu().double()
    want, mags = ds.cpu().double() @ cv, ds.cpu().double().abs() @ cv.abs()
    # exact products of bf16 planes in fp32 accumulators: at most 3 n / 16 sums in a row and 64 within and across
    # instructions and parts, each off by 2^-23; one rounding to the gradient's type
    tol = torch.finfo(dq.dtype).eps / 2 * want.abs() * 1.01 + (3 * n / 16 + 64) * 2.0 ** -23 * mags
    tol = tol + (2.0 ** -25 if dq.dtype == torch.float16 else 0.0)
    off = (dq.detach().cpu().double() - want).abs()
    assert bool((off <= tol).all()), float((off / tol).max())


SIZES = [(1, 1, 1), (1, 1000, 60), (2, 17, 128), (5, 3001, 256), (16, 64, 130), (17, 129, 512), (33, 515, 90), (64, 1000, 128),
         (65, 66, 300), (100, 257, 1024), (129, 4099, 60), (300, 1025, 256), (513, 700, 129), (1030, 130, 64), (4, 70000, 33), (21, 300, 384),
         (22, 300, 384), (32, 900, 256), (33, 900, 256), (16, 333, 512), (16, 333, 513), (50, 2000, 128)]


@pytest.mark.parametrize("m,n,d", SIZES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_and_gradient(dev, m, n, d, dtype):
    cat, q, ds = score_case(dev, m, n, d, dtype, dtype, m + n + d)
    s = cat.scores(q)
    assert s.shape == (m, n) and s.dtype == dtype
    check_scores(cat, q, s)
    s.backward(ds.to(dev))
    assert q.grad.dtype == dtype
    check_dq(cat, q, ds, q.grad)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("out_dtype", DTYPES)
def test_result_types(dev, dtype, out_dtype):
    for m, n, d in ((3, 500, 130), (150, 300, 130)):
        cat, q, ds = score_case(dev, m, n, d, dtype, out_dtype)
        s = cat.scores(q, dtype=out_dtype)
        check_scores(cat, q, s)
        s.backward(ds.to(dev))
        check_dq(cat, q, ds, q.grad)


@pytest.mark.parametrize("m", [1, 20, 200])
def test_part_of_the_catalogue_and_layouts(dev, m):
    """count below the capacity (rows behind it hold NaN); queries with strides;
    batched queries; upstream gradients that are expanded or transposed."""
    cat, q, _ = score_case(dev, m, 333, 200, torch.float32, torch.float32)
    cat.write(torch.full((100, 200), float("nan"), device=dev), start=233)
    for n in (0, 1, 150, 233):
        s = cat.scores(q, count=n)
        assert s.shape == (m, n)
        check_scores(cat, q, s, n)
        q.grad = None
        s.sum().backward()  # an expanded gradient
        check_dq(cat, q, torch.ones(m, n), q.grad, n)
        if n:
            ds = torch.randn(n, m)
            q.grad = None
            cat.scores(q, count=n).backward(ds.to(dev).t())
            check_dq(cat, q, ds.t(), q.grad, n)
            wide = torch.randn(m, n + 5)
            q.grad = None
            torch.autograd.backward([cat.scores(q, count=n)], [wide.to(dev)[:, 2:n + 2]])
            check_dq(cat, q, wide[:, 2:n + 2], q.grad, n)
    wide = torch.zeros(m, 207, device=dev)
    wide[:, 5:205] = q.detach()
    a, b = cat.scores(wide[:, 5:205], count=233), cat.scores(q.detach(), count=233)
    assert torch.equal(a, b)
    b3 = cat.scores(q.detach().reshape(1, m, 200), count=233)
    assert torch.equal(b3[0], b)
    assert torch.equal(cat.scores(q.detach()[0], count=233), cat.scores(q.detach()[:1], count=233)[0])
    # queries share a row: the gradient of the broadcast one is the sum
    one = q.detach()[:1].clone().requires_grad_()
    ds = torch.randn(m, 233)
    cat.scores(one.expand(m, 200), count=233).backward(ds.to(dev))
    cv = cat.read()[:233].cpu().double()
    tol = (3 * 233 / 16 + 64 + m) * 2.0 ** -23 * (ds.double().abs() @ cv.abs()).sum(0)
    assert bool(((one.grad.cpu().double()[0] - (ds.double() @ cv).sum(0)).abs() <= tol).all())


@pytest.mark.parametrize("m", [2, 40, 300])
def test_nonfinite_values_stay_in_their_row(dev, m):
    cat, q, _ = score_case(dev, m, 400, 256, torch.float32, torch.float32)
    bad = torch.zeros(2, 256, device=dev)
    bad[0, 3], bad[1, 200] = float("nan"), float("inf")
    cat.write(bad, rows=torch.tensor([7, 300], device=dev))
    with torch.no_grad():
        q[1, 255] = float("inf")
    s = cat.scores(q.detach())
    want = torch.zeros(m, 400, dtype=torch.bool)
    want[:, 7] = want[:, 300] = want[1] = True
    assert torch.equal(torch.isnan(s).cpu(), want)
    # an upstream gradient that is zero there does not bring the catalogue's NaN in by itself: 0 * NaN is NaN in
    # the formula, in its column of the gradient only
    ds = torch.zeros(m, 400, device=dev)
    ds[0, 5] = 1.0
    cat.scores(q).backward(ds)
    nan = torch.zeros(m, 256, dtype=torch.bool)
    nan[:, 3] = nan[:, 200] = True
    assert torch.equal(torch.isnan(q.grad).cpu(), nan)
    # infinities in the upstream gradient follow the formula: inf * value, NaN only where a value is zero
    cat2, q2, _ = score_case(dev, m, 64, 128, torch.float32, torch.float32)
    ds = torch.zeros(m, 64, device=dev)
    ds[0, 9] = float("inf")
    cat2.scores(q2).backward(ds)
    row = cat2.read()[9]
    want = ds[0, 9] * row
    assert torch.equal(torch.isnan(q2.grad[0]), torch.isnan(want))
    assert torch.equal(q2.grad[0][row != 0], want[row != 0]) and torch.isfinite(q2.grad[1:]).all()


def test_scale_extremes(dev):
    """Scales far apart, scale bytes 0 and 255 in given storage, sums that cancel."""
    cat, q, _ = score_case(dev, 5, 40, 256, torch.float32, torch.float32)
    x = cat.read().cpu()
    x[:, :128] *= 2.0 ** 60
    x[3] *= 2.0 ** -80
    cat.write(x.to(dev))
    s = cat.scores(q)
    check_scores(cat, q, s)
    qq = q.detach().clone()
    qq[:, :128] *= 2.0 ** -60
    check_scores(cat, qq, cat.scores(qq))
    codes, scales = cat.codes.clone(), cat.scales.clone()
    scales[0], scales[1] = 0, 255
    other = EmbeddingCatalogue.from_storage(codes, scales, 256)
    r = other.read()
    assert torch.isfinite(r[0]).all() and torch.isnan(r[1]).all()
    s = other.scores(q.detach())
    assert torch.isfinite(s[:, 0]).all() and torch.isnan(s[:, 1]).all() and torch.isfinite(s[:, 2:]).all()


def test_repeatable(dev):
    for m, n in ((1, 50000), (40, 50000), (700, 9000)):
        cat, q, ds = score_case(dev, m, n, 128, torch.float32, torch.float32)
        ds = ds.to(dev)
        runs = []
        for _ in range(3):
            s = cat.scores(q)
            runs.append((s.detach(), torch.autograd.grad(s, q, ds)[0]))
        assert all(torch.equal(a, runs[0][0]) and torch.equal(b, runs[0][1]) for a, b in runs)


@pytest.mark.parametrize("m,d", [(1, 100), (24, 100), (300, 100), (20, 200), (300, 300)])
def test_captured_together(dev, m, d):
    """A training step against the catalogue in one graph -- indexed write,
    scores, softmax loss, gradient -- replayed with eager work between; two
    graphs of the same catalogue alternate."""
    n = 700
    cat, q, _ = score_case(dev, m, n, d, torch.float32, torch.float32)
    new = torch.randn(30, d, device=dev)
    rows = torch.randint(0, n, (30,), device=dev)
    label = torch.randint(0, n, (m,), device=dev)

    def step(x):
        cat.write(new, rows=rows)
        s = cat.scores(x)
        loss = torch.logsumexp(s, 1) - s.gather(1, label[:, None])[:, 0]
        return s.detach(), torch.autograd.grad(loss, x, torch.ones_like(loss))[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    qs = [q, q.detach().flip(0).clone().requires_grad_()]
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for x in qs:
            step(x)
    torch.cuda.current_stream().wait_stream(side)
    for x in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(x))
        graphs.append(g)
    for k in range(4):
        new.copy_(torch.randn(30, d))
        rows.copy_(torch.randint(0, n, (30,)))
        for i in (k % 2, 1 - k % 2):
            graphs[i].replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in outs[i]]
            want = step(qs[i])
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), (k, i)


def test_another_stream(dev):
    cat, q, ds = score_case(dev, 50, 3000, 128, torch.bfloat16, torch.bfloat16)
    want = cat.scores(q)
    wg = torch.autograd.grad(want, q, ds.to(dev))[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = EmbeddingCatalogue(3000, 128, device=dev)
        again.write(cat.read())
        got = again.scores(q)
        gg = torch.autograd.grad(got, q, ds.to(dev))[0]
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want) and torch.equal(gg, wg)


def test_training_against_the_catalogue_and_adamw(dev):
    """Catalogue, scores, gradient and optimizer as they are used together."""
    from ceo_firm_matching import AdamW
    torch.manual_seed(0)
    n, d = 500, 60
    target = torch.nn.functional.normalize(torch.randn(n, d, device=dev), dim=1)
    cat = EmbeddingCatalogue(n, d, device=dev)
    cat.write(target)
    net = torch.nn.Linear(16, d).to(dev)
    opt = AdamW(net.parameters(), lr=1e-2, state_bits=8)
    x = torch.randn(128, 16, device=dev)
    label = torch.randint(0, n, (128,), device=dev)
    for _ in range(3):
        opt.zero_grad()
        q = torch.nn.functional.normalize(net(x), dim=1)
        loss = torch.nn.functional.cross_entropy(cat.scores(q) * 10, label)
        loss.backward()
        ref = torch.nn.functional.normalize(torch.nn.functional.linear(x, w := net.weight.detach().clone().requires_grad_(),
                                                                       net.bias.detach()), dim=1)
        torch.nn.functional.cross_entropy((ref @ cat.read().t()) * 10, label).backward()
        # the queries' e4m3 rounding moves each score by at most 2^-4 |q| |c|, the softmax's weights by 10 times that
        rel = float((net.weight.grad - w.grad).norm() / w.grad.norm())
        assert rel < 10 * 2.0 ** -4, rel
        opt.step()
    assert all(torch.isfinite(p).all() for p in net.parameters())


def test_offsets_past_32_bits(dev):
    """A catalogue of more than 2^32 bytes; scores and upstream gradients of
    more than 2^32 bytes: values at both ends."""
    n, d = 17_000_003, 256
    cat = EmbeddingCatalogue(n, d, device=dev)
    x = torch.nn.functional.normalize(torch.randn(200, d, device=dev), dim=1)
    cat.write(x[:100])
    cat.write(x[100:], start=n - 100)
    assert torch.equal(cat.read(start=n - 100), cat.read(rows=torch.arange(n - 100, n, device=dev)))
    small = EmbeddingCatalogue(200, d, device=dev)
    small.write(x)
    assert torch.equal(cat.read(start=n - 100), small.read(start=100))
    q = torch.nn.functional.normalize(torch.randn(130, d, device=dev), dim=1).bfloat16()
    want = small.scores(q)
    for m in (1, 20, 130):  # 130 x n in bf16 is 4.4e9 bytes
        qm = q[:m].clone().requires_grad_()
        s = cat.scores(qm)
        # few and many queries sum in other orders: each is within its own bound of the exact score
        for part, ref in ((s[:, :100], want[:m, :100]), (s[:, n - 100:], want[:m, 100:])):
            assert float((part.detach().float() - ref.float()).abs().max()) <= 2 * (2.0 ** -8 + 2.0 ** -10)  # |scores| <= 1: half a step of bf16
        assert not s[:, 100:n - 100:100003].any()
        ds = torch.zeros(m, n, dtype=torch.bfloat16, device=dev)
        ds[:, :100], ds[:, n - 100:] = 0.5, -0.25
        g = torch.autograd.grad(s, qm, ds)[0]
        v = small.read().double()
        row = 0.5 * v[:100].sum(0) - 0.25 * v[100:].sum(0)
        tol = 2.0 ** -8 * row.abs() * 1.01 + (200 + 64) * 2.0 ** -23 * v.abs().sum(0)
        assert bool(((g.double() - row).abs() <= tol).all())
        del s, ds, g


@pytest.mark.parametrize("n", [64, 65, 127, 128, 129, 191, 193, 257, 511, 513])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_of_odd_length_read_no_neighbour(dev, n, dtype):
    """The gradient of 16-bit rows at odd distances, next to NaN in front of,
    between and behind the rows."""
    for m in (2, 33, 130):
        cat, q, ds = score_case(dev, m, n, 96, dtype, dtype, n)
        want = torch.autograd.grad(cat.scores(q), q, ds.to(dev))[0]
        for before, gap in ((0, 0), (0, 2), (2, 2), (1, 1), (1, 2), (4, 3)):
            store = torch.full((before + m * (n + gap) + 2,), float("nan"), dtype=dtype, device=dev)
            view = store[before:before + m * (n + gap)].view(m, n + gap)[:, :n]
            view.copy_(ds)
            got = torch.autograd.grad(cat.scores(q), q, view)[0]
            assert torch.equal(got, want), (m, before, gap)


def test_empty_calls(dev):
    empty = EmbeddingCatalogue(0, 5, device=dev)
    empty.write(torch.zeros(2, 5, device=dev), rows=torch.tensor([0, -1], device=dev))
    q = torch.ones(2, 5, device=dev, requires_grad=True)
    s = empty.scores(q)
    assert s.shape == (2, 0) and not empty.read(rows=torch.tensor([0], device=dev)).any()
    s.sum().backward()
    assert not q.grad.any()
    cat = EmbeddingCatalogue(7, 5, device=dev)
    none = torch.zeros(0, 5, device=dev, requires_grad=True)
    cat.write(none)
    cat.write(none, rows=torch.zeros(0, dtype=torch.int64, device=dev))
    s = cat.scores(none)
    assert s.shape == (0, 7) and cat.read(rows=torch.zeros(0, dtype=torch.int64, device=dev)).shape == (0, 5)
    s.sum().backward()
    assert none.grad.shape == (0, 5)
