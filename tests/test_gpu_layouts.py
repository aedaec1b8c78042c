"""GPU checks of operands that lie badly in memory: off 16 bytes, with odd strides, one well and the other not."""

import pytest
import torch

from test_gpu_linear_loss import dev, inputs, plain, within  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def lying(t, how):
    """A copy of the matrix t that lies so: well, one element off 16 bytes, or with an odd stride."""
    if how == "well":
        return t.clone()
    if how == "off":
        return torch.zeros(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape).copy_(t)
    return torch.zeros(t.shape[0], t.shape[1] + 1, dtype=t.dtype, device=t.device)[:, :-1].copy_(t)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,H,V", [(5, 64, 300), (100, 128, 3000), (129, 64, 7), (400, 128, 3000), (400, 64, 9000), (511, 256, 100),
                                   (2100, 64, 500)])
def test_loss(dev, N, H, V, dtype):
    """The same bits however x and the weight lie."""
    from linear_loss import linear_cross_entropy
    print("layouts", N, H, V, dtype, flush=True)
    x, w, t, d = inputs(dev, N, H, V, dtype, N + V)
    want, tol = plain(x, w, t, d)
    first = None
    for a in ("well", "off", "odd"):
        for b in ("well", "off", "odd"):
            X, W = lying(x, a).requires_grad_(True), lying(w, b).requires_grad_(True)
            loss = linear_cross_entropy(X, W, t, reduction="none")
            got = [loss.detach(), *torch.autograd.grad(loss, [X, W], d)]
            for g, c, e, what in zip(got, want, tol, ("loss", "dx", "dw")):
                within(g, c, e, (what, a, b))
            first = first or got
            assert all(torch.equal(g, f) for g, f in zip(got[1:], first[1:])) or dtype == torch.float32, (a, b)
            only = linear_cross_entropy(lying(x, a).requires_grad_(True), lying(w, b), t, reduction="none")
            assert torch.equal(only.detach(), got[0])
