"""The 8-bit embedding catalogue on the CPU: quantised values, scores and the
queries' gradient against the definition, and what is refused (also by the
C-ABI)."""
import numpy as np
import pytest
import torch

from ceo_firm_matching import EmbeddingCatalogue
from ceo_firm_matching import _native as N
from ceo_firm_matching import block8


def exact_e4m3(x):
    """Rows in 64 bits as their e4m3 blocks hold them (finite values)."""
    m, d = x.shape
    b = torch.nn.functional.pad(x.double(), (0, -d % 128)).reshape(m, -1, 128)
    big = b.abs().amax(2, keepdim=True)
    e = torch.full_like(big, -100.0)
    for k in range(-100, 121):
        e = torch.where(448 * 2.0 ** (k - 1) < big, torch.full_like(e, float(k)).clamp_min(-100), e)
    y = b / torch.exp2(e)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(y / step) * step * torch.exp2(e)).reshape(m, -1)[:, :d]


def rows_of(m, d, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(m, d, generator=g) * torch.exp(3 * torch.randn(m, 1, generator=g))).to(dtype)


@pytest.mark.parametrize("d", [1, 60, 128, 129, 300])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_written_rows_read_back_as_defined(d, dtype):
    x = rows_of(9, d, d, dtype)
    cat = EmbeddingCatalogue(20, d)
    cat.write(x, start=5)
    got = cat.read()
    assert torch.equal(got[5:14].double(), exact_e4m3(x))
    assert not got[:5].any() and not got[14:].any()
    assert torch.equal(cat.read(start=5, count=9, dtype=torch.bfloat16).float(), got[5:14])  # bf16 holds every value
    assert torch.equal(cat.read(rows=torch.tensor([13, -1, 5, 20, 13])),
                       torch.stack([got[13], 0 * got[0], got[5], 0 * got[0], got[13]]))


def test_all_codes_scales_and_edges():
    """Every e4m3 value at several scales; the border of a scale; tiny, huge,
    zero, infinite and NaN values."""
    v = torch.arange(256).to(torch.uint8).view(torch.float8_e4m3fn).float()
    v = v[torch.isfinite(v)]
    v = torch.cat([v, torch.full((256 - v.numel(),), 448.0)]).reshape(2, 128)
    v[0, 0] = 448.0
    for e in (-100, -30, 0, 50, 119):
        cat = EmbeddingCatalogue(2, 128)
        cat.write(v * 2.0 ** e)
        assert torch.equal(cat.read(), v * 2.0 ** e) and (cat.scales == 127 + e).all()
    up = torch.zeros(1, 128)
    up[0, 0] = float(np.nextafter(np.float32(448), np.float32(500)))
    cat = EmbeddingCatalogue(1, 128)
    cat.write(up)
    assert int(cat.scales) == 128 and float(cat.read()[0, 0]) == 448.0
    x = torch.zeros(4, 128)
    x[0, 3], x[0, 4], x[1, 0], x[2, :2] = float("inf"), 2.0, float("nan"), torch.tensor([3e38, -1e-38])
    x[3, 5] = 1e-45
    cat = EmbeddingCatalogue(4, 128)
    cat.write(x)
    r = cat.read()
    assert torch.isnan(r[0, 3]) and float(r[0, 4]) == 2.0 and torch.isnan(r[1, 0]) and float(r[1, 1]) == 0.0
    assert abs(float(r[2, 0]) / 3e38 - 1) <= 2.0 ** -4 and not r[3].any()


def test_rows_named_twice_take_the_last_and_strays_are_left_out():
    x = rows_of(6, 70, 3)
    cat = EmbeddingCatalogue(4, 70)
    cat.write(x, rows=torch.tensor([2, -1, 2, 4, 0, 2]))
    want = torch.zeros(4, 70, dtype=torch.float64)
    want[2], want[0] = exact_e4m3(x)[5], exact_e4m3(x)[4]
    assert torch.equal(cat.read().double(), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_scores_and_gradient(dtype):
    d, n = 200, 37
    cat = EmbeddingCatalogue(n + 3, d)
    c = torch.nn.functional.normalize(rows_of(n + 3, d, 1), dim=1)
    cat.write(c)
    q = torch.nn.functional.normalize(rows_of(5, d, 2), dim=1).to(dtype).requires_grad_()
    s = cat.scores(q, count=n)
    cv = cat.read()[:n].double()
    qv = exact_e4m3(q.detach())
    eps = torch.finfo(dtype).eps / 2
    mags = qv.abs() @ cv.abs().t()
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    assert s.dtype == dtype
    assert bool(((s.double() - qv @ cv.t()).abs() <= eps * s.double().abs() * 1.01 + (d + 2) * 2.0 ** -24 * mags + tiny).all())
    ds = torch.randn(5, n).to(dtype)
    s.backward(ds)
    want, mags = ds.double() @ cv, ds.double().abs() @ cv.abs()
    assert q.grad.dtype == dtype
    assert bool(((q.grad.double() - want).abs() <= eps * want.abs() * 1.01 + (n + 2) * 2.0 ** -24 * mags + tiny).all())


def test_gradient_against_differences():
    """Where a query and its moved copies are values e4m3 holds, scores are
    linear in it: their differences are the gradient."""
    d, n = 130, 11
    cat = EmbeddingCatalogue(n, d)
    cat.write(rows_of(n, d, 4))
    q = torch.randint(-7, 8, (1, d)).float()
    q[0, 0] = q[0, 129] = 15.0  # both blocks keep their scale 2^-4 ... and every integer to 15 is held
    q.requires_grad_()
    ds = torch.randn(1, n)
    cat.scores(q).backward(ds)
    for k in (1, 64, 128):
        lo, hi = q.detach().clone(), q.detach().clone()
        lo[0, k] -= 1
        hi[0, k] += 1
        diff = ((cat.scores(hi).double() - cat.scores(lo).double()) * ds.double()).sum() / 2
        scale = float((cat.scores(hi).double().abs() * ds.double().abs()).sum()) + abs(float(diff))
        assert abs(float(diff) - float(q.grad[0, k])) <= (2 * d + n) * 2.0 ** -24 * scale * 8


def test_shapes_views_and_empty_calls():
    cat = EmbeddingCatalogue(6, 33)
    x = rows_of(6, 33, 7)
    wide = torch.zeros(6, 50)
    wide[:, 10:43] = x
    cat.write(wide[:, 10:43])
    assert torch.equal(cat.read().double(), exact_e4m3(x))
    cat.write(x.t().contiguous().t())
    assert torch.equal(cat.read().double(), exact_e4m3(x))
    assert cat.scores(x[0]).shape == (6,) and cat.scores(x.reshape(2, 3, 33)).shape == (2, 3, 6)
    assert cat.scores(x[:0]).shape == (0, 6) and cat.scores(x, count=0).shape == (6, 0)
    cat.write(x[:0])
    cat.write(x[:0], rows=torch.zeros(0, dtype=torch.int64))
    assert cat.read(count=0).shape == (0, 33)
    empty = EmbeddingCatalogue(0, 5)
    empty.write(torch.zeros(2, 5), rows=torch.tensor([0, -1]))
    assert empty.scores(torch.zeros(2, 5)).shape == (2, 0) and not empty.read(rows=torch.tensor([0])).any()
    other = EmbeddingCatalogue.from_storage(cat.codes, cat.scales, 33)
    assert torch.equal(other.read(), cat.read())
    s = cat.scores(x.clone().requires_grad_())
    cat.write(x[:1])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        s.sum().backward()  # the rows it was computed with are gone


def test_refusals():
    cat = EmbeddingCatalogue(4, 8)
    x = torch.zeros(2, 8)
    for call in (lambda: EmbeddingCatalogue(-1, 8), lambda: EmbeddingCatalogue(4, 0), lambda: cat.write(torch.zeros(2, 9)),
                 lambda: cat.write(x, start=3), lambda: cat.write(x, start=-1), lambda: cat.write(torch.zeros(8)),
                 lambda: cat.write(x, rows=torch.zeros(3, dtype=torch.int64)), lambda: cat.write(x, rows=torch.zeros(2)),
                 lambda: cat.write(x, rows=torch.zeros(2, dtype=torch.int64), start=1), lambda: cat.read(start=5),
                 lambda: cat.read(start=1, count=4), lambda: cat.read(rows=torch.zeros(1, dtype=torch.int64), count=1),
                 lambda: cat.scores(torch.zeros(2, 7)), lambda: cat.scores(x, count=5), lambda: cat.scores(x, count=-1),
                 lambda: EmbeddingCatalogue.from_storage(cat.codes, cat.scales, 129),
                 lambda: EmbeddingCatalogue.from_storage(cat.codes.float(), cat.scales, 8),
                 lambda: EmbeddingCatalogue.from_storage(cat.codes[:, :64], cat.scales, 8),
                 lambda: EmbeddingCatalogue.from_storage(cat.codes, cat.scales[:3], 8)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: cat.write(x.double()), lambda: cat.read(dtype=torch.float64), lambda: cat.scores(x.long()),
                 lambda: cat.scores(x, dtype=torch.float64)):
        with pytest.raises(NotImplementedError):
            call()


def test_host_argument_errors():
    """tt_cat_*: decided on the host before anything is enqueued."""
    L = N.lib()
    buf = np.zeros(1 << 16, dtype=np.float32)
    p = buf.ctypes.data

    def write(x=p, dt=0, m=2, ldx=8, d=8, rows=None, row0=0, codes=p, scales=p, cap=4, owner=p):
        return L.tt_cat_write(x, dt, m, ldx, d, rows, row0, codes, scales, cap, owner, None)

    assert write(m=0) == N.TT_OK
    for kw in (dict(x=None), dict(dt=3), dict(m=-1), dict(ldx=7), dict(d=0), dict(d=1 << 21), dict(row0=3), dict(row0=-1),
               dict(codes=None), dict(scales=None), dict(cap=-1), dict(rows=p, owner=None), dict(rows=p, m=2 ** 31), dict(x=p + 2), dict(rows=p + 4),
               dict(m=2 ** 41, cap=2 ** 41)):
        assert write(**kw) == N.TT_ERR_ARG, kw

    def read(codes=p, scales=p, cap=4, d=8, rows=None, row0=0, m=2, out=p, dt=0, ldo=8):
        return L.tt_cat_read(codes, scales, cap, d, rows, row0, m, out, dt, ldo, None)

    assert read(m=0) == N.TT_OK
    for kw in (dict(codes=None), dict(out=None), dict(dt=-1), dict(ldo=7), dict(row0=3), dict(m=5), dict(d=0)):
        assert read(**kw) == N.TT_ERR_ARG, kw

    def scores(q=p, dt=0, m=2, ldq=8, d=8, codes=p, scales=p, n=4, out=p, odt=0, ws=p, wsb=1 << 16):
        return L.tt_cat_scores(q, dt, m, ldq, d, codes, scales, n, out, odt, ws, wsb, None)

    assert scores(m=0) == N.TT_OK and scores(n=0) == N.TT_OK
    for kw in (dict(q=None), dict(dt=5), dict(odt=5), dict(ldq=7), dict(codes=None), dict(scales=None), dict(out=None),
               dict(d=0), dict(m=-2), dict(n=-1), dict(q=p + 1, dt=1), dict(out=p + 2), dict(codes=p + 8)):
        assert scores(**kw) == N.TT_ERR_ARG, kw
    assert L.tt_cat_scores_workspace_bytes(-1, 4, 8) == N.TT_ERR_ARG
    need = L.tt_cat_scores_workspace_bytes(70, 4, 8)
    assert need > 0 and scores(m=70, wsb=need - 1) == N.TT_ERR_WORKSPACE and scores(m=70, ws=None, wsb=need) == N.TT_ERR_ARG
    assert scores(m=70, ws=p + 8, wsb=need) == N.TT_ERR_ARG
    assert L.tt_cat_dq_workspace_bytes(4, 4, 0, 0) == N.TT_ERR_ARG

    def dq(ds=p, dt=0, m=2, lds=4, n=4, codes=p, scales=p, d=8, out=p, odt=0, ws=p, wsb=1 << 30):
        return L.tt_cat_dq(ds, dt, m, lds, n, codes, scales, d, out, odt, ws, wsb, None)

    assert dq(m=0) == N.TT_OK
    for kw in (dict(ds=None), dict(dt=7), dict(odt=7), dict(lds=3), dict(codes=None), dict(out=None), dict(d=0), dict(n=-1),
               dict(codes=p + 8), dict(ds=p + 2), dict(out=p + 1, odt=1)):
        assert dq(**kw) == N.TT_ERR_ARG, kw


def test_inference_mode():
    with torch.inference_mode():
        cat = EmbeddingCatalogue(3, 5)
        cat.write(torch.ones(3, 5))
        assert torch.equal(cat.scores(torch.ones(2, 5)), torch.full((2, 3), 5.0))


def test_block_scale_is_the_smallest_that_fits():
    for amax, e in ((448.0, 0), (449.0, 1), (1.75, -8), (1.7500001, -7), (2.0 ** -110, -100), (0.0, -100)):
        x = torch.zeros(1, 128)
        x[0, 9] = amax
        _, s = block8.encode(x)
        assert int(s) - 127 == e, amax
