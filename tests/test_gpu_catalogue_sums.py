"""Scores whose products cancel: sums in 32 bits, rounded once, whatever the
results' type."""
import pytest
import torch

from ceo_firm_matching import EmbeddingCatalogue

pytestmark = pytest.mark.gpu


@pytest.fixture
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    return torch.device("cuda:0")


def cancelling(m, n, d, seed):
    """Rows of e4m3 values (scale 1 in every block): two large products of each
    block cancel, within 8 neighbours; the others are small and of one sign."""
    g = torch.Generator().manual_seed(seed)
    small = torch.tensor([0.25, 0.34375, 0.40625, 0.46875, 0.5625, 0.6875, 0.8125, 0.9375])
    q, c = (small[torch.randint(0, 8, (r, d), generator=g)] for r in (m, n))
    for b in range(0, d, 128):
        i, j = (b + 8 * int(torch.randint(0, min(128, d - b) // 8, (), generator=g)) + torch.randperm(8, generator=g)[:2]).tolist()
        q[:, i] = q[:, j] = c[:, i] = 448.0
        c[:, j] = -448.0
    return q, c


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,n,d", [(1, 700, 128), (16, 333, 512), (20, 130, 256), (24, 260, 384), (30, 200, 512), (40, 1000, 128),
                                   (64, 300, 256), (50, 300, 300), (65, 129, 128), (300, 400, 256), (130, 257, 1000)])
def test_products_that_cancel(dev, m, n, d, dtype):
    q, c = cancelling(m, n, d, m + n + d)
    cat = EmbeddingCatalogue(n, d, device=dev)
    cat.write(c.to(dev))
    assert torch.equal(cat.read().cpu(), c)  # e4m3 holds the values: the queries' rounding is none either
    s = cat.scores(q.to(dev), dtype=dtype).cpu().double()
    want = q.double() @ c.double().t()
    # products are exact in 32 bits, each sum (cut off, not rounded, allowed for) is off by 2^-23 of what was added up:
    # the large products of a block meet in one matrix instruction of 32, at most 33 sums; outside it only the small
    # ones count; then one rounding to the type
    tol = (torch.finfo(dtype).eps / 2 * want.abs() * 1.01 + 33 * 2.0 ** -23 * 2 * 448.0 ** 2 * -(-d // 128)
           + (d + 2) * 2.0 ** -23 * want.abs())
    off = (s - want).abs()
    assert bool((off <= tol).all()), float((off / tol).max())
