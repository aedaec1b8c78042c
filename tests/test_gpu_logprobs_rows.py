"""GPU checks of the log probabilities of rows that hold NaN and of targets outside the vocabulary, and of their gradients,
against plain 64-bit forms.

A row with a NaN logit has no log probability, entropy or gradient that is a number, whatever else it holds: its sum is NaN.
Rows of nothing but -inf (banned tokens) are something else: log probabilities -inf, entropy 0, no gradient.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import gdn_lib
    gdn_lib.load()
    return torch.device("cuda:0")


# a short row, one of part of a piece, one of whole pieces, one of whole pieces and a part
@pytest.mark.parametrize("V", [3, 300, 16384, 20001])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_nan(dev, V, dtype):
    from token_logprobs import token_logprobs
    z = torch.randn(9, V, device=dev)
    z[0] = math.nan                      # nothing but NaN
    z[1] = math.nan
    z[1, ::2] = -math.inf                # NaN and banned tokens, the target a NaN
    z[2] = -math.inf
    z[2, V - 1] = math.nan               # one NaN, the rest banned, the target banned
    z[3, V // 2] = math.nan              # one NaN among numbers
    z[4] = -math.inf                     # nothing left, no NaN
    z[6] = math.nan                      # ignored
    z[7] = math.inf
    z[7, 0] = math.nan
    z = z.to(dtype).requires_grad_(True)
    y = torch.tensor([0, 1, 0, 1, 2, 1, -100, 1, 2], device=dev)
    top = min(3, V)
    r = token_logprobs(z, y, entropy=True, top=top)
    odd = torch.tensor([0, 1, 2, 3, 7], device=dev)
    assert bool(r.logp[odd].isnan().all()) and bool(r.entropy[odd].isnan().all())
    assert bool(r.top_logp[odd].isnan().all())
    want = torch.sort(z.detach().double(), dim=-1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(r.top_ids, want)
    assert float(r.logp[4]) == -math.inf and float(r.entropy[4]) == 0.0 and bool((r.top_logp[4] == -math.inf).all())
    assert float(r.logp[6]) == 0.0 and bool(torch.isfinite(r.logp[[5, 8]]).all())
    plain = token_logprobs(z.detach(), y)  # the kernel without entropy and alternatives
    assert torch.equal(plain.logp.nan_to_num(nan=7.0), r.logp.nan_to_num(nan=7.0))
    for loss in ((r.logp,), (r.entropy,), (r.logp, r.entropy)):
        (dz,) = torch.autograd.grad(loss, [z], [torch.ones_like(x) for x in loss], retain_graph=True)
        assert bool(dz[odd].isnan().all()), len(loss)
        assert not bool(dz[4].any())
        assert bool(torch.isfinite(dz[[5, 8]]).all()) and bool(dz[[5, 8]].any(-1).all())
        if len(loss) == 1 and loss[0] is r.logp:
            assert not bool(dz[6].any())


@pytest.mark.parametrize("dtype", DTYPES)
def test_targets_outside_the_vocabulary(dev, dtype):
    """They make their own log probability NaN and the gradient of a loss that it is part of; the entropy of the row does not
    depend on its target, nor does the entropy's gradient.  Bound: as in the other tests of dlogits, a few 2^-23 of the terms
    (each below |x| + H < 40 times its probability) and the output's own rounding."""
    from token_logprobs import token_logprobs
    z = (3 * torch.randn(4, 9001, device=dev)).to(dtype).requires_grad_(True)
    y = torch.tensor([9001, -1, 7, -100], device=dev)
    w = torch.randn(4, device=dev)
    r = token_logprobs(z, y, entropy=True)
    assert r.logp.isnan().tolist() == [True, True, False, False] and bool(torch.isfinite(r.entropy).all())
    (dz,) = torch.autograd.grad([r.entropy], [z], [w], retain_graph=True)
    lp = torch.log_softmax(z.detach().double(), -1)
    p = lp.exp()
    H = -(p * lp).sum(-1, keepdim=True)
    want = -w.double()[:, None] * p * (lp + H)
    room = w.double().abs()[:, None] * p * 40 * 2 ** -16 + want.abs() * torch.finfo(dtype).eps / 2
    room = room + torch.finfo(dtype).smallest_normal
    assert bool(((dz.double() - want).abs() <= room).all())
    (dz,) = torch.autograd.grad([r.logp, r.entropy], [z], [w, w])
    assert bool(dz[:2].isnan().all()) and bool(torch.isfinite(dz[2:]).all())
