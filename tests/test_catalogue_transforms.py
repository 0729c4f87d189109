"""Forward-mode derivatives, function transforms and tracing of the catalogue's
calls: right or refused, never dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from ceo_firm_matching import EmbeddingCatalogue

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]


def make(name):
    if name != "cpu" and not torch.cuda.is_available():
        pytest.skip("no HIP device")
    g = torch.Generator().manual_seed(0)
    cat = EmbeddingCatalogue(9, 20, device=name)
    cat.write(torch.randn(9, 20, generator=g).to(name))
    return cat, torch.randn(3, 20, generator=g).to(name), torch.randn(3, 20, generator=g).to(name)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("shape", [(3, 20), (1, 3, 20), (20,)])
def test_forward_mode_is_refused(device, requires_grad, grad_mode, shape):
    cat, q, t = make(device)
    q, t = (x[:1].reshape(shape) if shape == (20,) else x.reshape(shape) for x in (q, t))
    with fwad.dual_level(), torch.set_grad_enabled(grad_mode):
        dual = fwad.make_dual(q.requires_grad_(requires_grad), t)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            cat.scores(dual)
        # the level alone changes nothing for queries without a tangent
        assert torch.equal(cat.scores(q).detach(), cat.scores(q.detach()))
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(cat.scores, (q.detach(),), (t,))


@pytest.mark.parametrize("device", DEVICES)
def test_reverse_mode_is_what_it_was(device):
    cat, q, t = make(device)
    q.requires_grad_()
    s = cat.scores(q)
    ds = torch.ones_like(s)
    s.backward(ds)
    assert torch.allclose(q.grad, ds @ cat.read(), rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
def test_tracing_is_refused_on_the_device():
    """A traced graph would hold the empty result and no launch."""
    cat, q, _ = make("cuda:0")
    rows = torch.tensor([1, 2, 3], device="cuda:0")
    for call in (lambda x: cat.scores(x), lambda x: cat.read(rows=rows) + x, lambda x: (cat.write(x, rows=rows), x + 1)[1]):
        with pytest.raises(NotImplementedError, match="trac"):
            torch.jit.trace(call, (q,), check_trace=False)
    assert cat.scores(q).shape == (3, 9)
