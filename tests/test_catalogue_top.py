"""Values next to float32's largest: held as finite ones, within 2^-4."""
import pytest
import torch

from ceo_firm_matching import EmbeddingCatalogue

TOP = torch.finfo(torch.float32).max


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [False, True])
def test_largest_values(device, dtype, rows):
    if device != "cpu" and not torch.cuda.is_available():
        pytest.skip("no HIP device")
    v = torch.tensor([1.0, 1.74, 1.75, 1.76, 1.86, 1.875, 1.9, 1.937, 1.9375, 1.94, 1.99], dtype=torch.float64) * 2.0 ** 127
    v = torch.cat([v.float(), torch.tensor([TOP])]).to(dtype)
    v = v[torch.isfinite(v)]
    # one large value a row, its negative, and a row that an infinity shares
    x = torch.zeros(3 * v.numel(), 130, dtype=dtype)
    n = v.numel()
    x[:n, 0], x[n:2 * n, 129], x[2 * n:, 3], x[2 * n:, 4] = v, -v, v, float("inf")
    cat = EmbeddingCatalogue(3 * n, 130, device=device)
    cat.write(x.to(device), rows=torch.arange(3 * n, device=device) if rows else None)
    got = cat.read().cpu()
    assert torch.isnan(got[2 * n:, 4]).all()
    got[2 * n:, 4] = 0
    want = torch.where(torch.isfinite(x), x, torch.zeros_like(x)).double()
    assert torch.isfinite(got).all()
    assert bool(((got.double() - want).abs() <= 2.0 ** -4 * want.abs()).all())
    # as queries: their own inner products with a unit vector
    unit = EmbeddingCatalogue(1, 130, device=device)
    unit.write(torch.eye(130, device=device)[:1])
    s = unit.scores(x[:n].to(device), dtype=torch.float32).cpu()[:, 0]
    assert torch.equal(s, got[:n, 0])
