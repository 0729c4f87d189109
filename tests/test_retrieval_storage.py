"""retrieval_ranks(storage=...): both storages take and refuse the same calls."""
import pytest
import torch

from ceo_firm_matching import contrastive

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("storage", [None, "e4m3"])
def test_fewer_candidates_than_firms_are_refused(device, storage):
    if device != "cpu" and not torch.cuda.is_available():
        pytest.skip("no HIP device")
    g = torch.Generator().manual_seed(0)
    f = torch.nn.functional.normalize(torch.randn(8, 12, generator=g), dim=1).to(device)
    for cap in (None, 7):
        with pytest.raises(ValueError, match="must map onto"):
            contrastive.retrieval_ranks(f, f[:5], cap=cap, storage=storage)
    # a cap that leaves as many, and more candidates than firms: the first min(firms, cap) pairs
    for cap, c in ((5, f[:5]), (None, torch.cat([f, -f])), (3, torch.cat([f, -f]))):
        ranks = contrastive.retrieval_ranks(f, c, cap=cap, storage=storage)
        assert ranks.tolist() == [1] * min(8, cap or 8)
