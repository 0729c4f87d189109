"""The package's own paths through AdamW and the 8-bit catalogue:
train_contrastive(optimizer=...), retrieval_ranks(storage=...),
compute_retrieval_metrics(storage=...)."""
import pytest
import torch

from test_contrastive_train import _cfg, _data
from ceo_firm_matching import EmbeddingCatalogue, block8, contrastive

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]


def _dev(name):
    if name != "cpu" and not torch.cuda.is_available():
        pytest.skip("no HIP device")
    return torch.device(name)


def _train(dev, **kw):
    from torch.utils.data import DataLoader
    from ceo_firm_matching.data import CEOFirmDataset
    data, meta = _data()
    torch.manual_seed(77)
    loader = DataLoader(CEOFirmDataset(data), batch_size=128, shuffle=True)
    return contrastive.train_contrastive(loader, loader, meta, _cfg(dev), **kw)


@pytest.mark.parametrize("device", DEVICES)
def test_train_contrastive_with_adamw(device, monkeypatch):
    dev = _dev(device)
    got = _train(dev, optimizer="adamw", weight_decay=0.02)
    with monkeypatch.context() as mp:
        mp.setattr(contrastive, "AdamW", lambda ps, lr, weight_decay, state_bits: torch.optim.AdamW(ps, lr=lr, weight_decay=weight_decay))
        want = _train(dev, optimizer="adamw", weight_decay=0.02)
    lr, steps = 4e-4, 14
    far = 0
    for (k, a), b in zip(got.named_parameters(), want.parameters()):
        d = (a - b).detach().abs()
        # a gradient near zero that differs by its last bits moves a value by up to 2 lr a step, another way each
        # time; such values are few, all others stay within the rounding of 14 updates
        assert float(d.max()) <= 2 * lr * steps, k
        far += int((d > 1e-2 * lr * steps).sum()) if not k.endswith((".0.bias", ".4.bias")) else 0
    assert far <= 0.02 * sum(p.numel() for p in got.parameters())
    eight = _train(dev, optimizer="adamw8bit")
    assert all(torch.isfinite(p).all() for p in eight.parameters())
    with pytest.raises(ValueError, match="optimizer"):
        _train(dev, optimizer="sgd")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("m,n,d", [(1, 1, 8), (50, 50, 30), (257, 400, 128)])
def test_ranks_by_the_catalogue(device, m, n, d):
    dev = _dev(device)
    g = torch.Generator().manual_seed(m + n)
    ce = torch.nn.functional.normalize(torch.randn(n, d, generator=g), dim=1)
    row0 = n - m
    fe = torch.nn.functional.normalize(ce[row0:] + 0.3 * torch.randn(m, d, generator=g), dim=1)
    cat = EmbeddingCatalogue(n, d, device=dev)
    cat.write(ce.to(dev))
    ranks = contrastive.catalogue_ranks(fe.to(dev), cat, row0).cpu()
    assert ranks.dtype == torch.int32
    s = block8.decode(*block8.encode(fe), d).double() @ cat.read().cpu().double().t()
    own = s.gather(1, torch.arange(row0, n)[:, None])
    near = (d + 2) * 2.0 ** -23  # |q| |c| <= 1.1, sums in 32 bits
    lo, hi = (s > own + 2 * near).sum(1) + 1, (s > own - 2 * near).sum(1)
    assert bool((ranks >= lo).all()) and bool((ranks <= hi).all())
    if m == n:
        assert torch.equal(contrastive.retrieval_ranks(fe.to(dev), ce.to(dev), cap=None, storage="e4m3").cpu(), ranks)
    with pytest.raises(ValueError):
        contrastive.catalogue_ranks(fe.to(dev), cat, row0 + 1)
    with pytest.raises(ValueError):
        contrastive.retrieval_ranks(fe, ce, storage="int4")


@pytest.mark.parametrize("device", DEVICES)
def test_retrieval_metrics_with_8_bit_storage(device):
    dev = _dev(device)
    data, meta = _data()
    cfg = _cfg(dev)
    torch.manual_seed(1)
    model = contrastive.ContrastiveCEOFirmMatcher(meta, cfg).to(dev)
    a = contrastive.compute_retrieval_metrics(model, data, cfg)
    b = contrastive.compute_retrieval_metrics(model, data, cfg, storage="e4m3")
    assert set(a) == set(b) and all(0 <= b[k] <= 1 for k in b if k != "median_rank")
