"""GPU checks that forward-mode tangents are refused, forward and backward, and that an open level alone changes nothing."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import gdn_lib
    gdn_lib.load()
    return torch.device("cuda:0")


def test_operators_at_both_ends(dev):
    import mxfp4
    from embedding import Embedding, embedding
    from linear_loss import linear_cross_entropy
    g = torch.Generator(device=dev)
    g.manual_seed(0)
    x, w = torch.randn(6, 64, device=dev, generator=g), torch.randn(9, 64, device=dev, generator=g)
    t = torch.randint(0, 9, (6,), device=dev, generator=g)
    q, table = mxfp4.quantize(w), Embedding(9, 64, device=dev)
    for call, at, out in ((lambda a: linear_cross_entropy(a, w, t, reduction="none"), x, (6,)),
                          (lambda a: linear_cross_entropy(x, a, t, reduction="none"), w, (6,)),
                          (lambda a: embedding(t, a), w, (6, 64)), (lambda a: mxfp4.linear(a, q), x, (6, 9))):
        want = call(at)
        d = torch.randn(out, device=dev, generator=g)
        leaf = at.clone().requires_grad_(True)
        grad, = torch.autograd.grad(call(leaf), leaf, d)
        with fwAD.dual_level():
            assert torch.equal(call(at), want)
            assert torch.equal(torch.autograd.grad(call(leaf), leaf, d)[0], grad)
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call(fwAD.make_dual(at, torch.ones_like(at)))
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                torch.autograd.grad(call(leaf), leaf, fwAD.make_dual(d, d))
        assert torch.equal(call(at), want)
    weight = table.weight.detach()
    with fwAD.dual_level(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
        torch.func.functional_call(table, {"weight": fwAD.make_dual(weight, weight)}, (t,))
