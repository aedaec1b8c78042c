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


def test_last_tokens_of_long_sequences(dev):
    """hidden[:, -1]: rows more than 8 MiB apart, with gradients, through a head and a 4-bit weight; and a head of such rows."""
    import mxfp4
    from linear_loss import linear_cross_entropy
    B, T, H, V = 70, 4097, 1024, 300
    hidden = torch.zeros(B, T, H, dtype=torch.bfloat16, device=dev)
    x, w, t, d = inputs(dev, B, H, V, torch.bfloat16, 3)
    hidden[:, -1] = x
    far = hidden[:, -1].detach().requires_grad_(True)
    assert far.stride(0) * 2 > 1 << 23
    near, w = x.requires_grad_(True), w.requires_grad_(True)
    got, want = (linear_cross_entropy(a, w, t, reduction="none") for a in (far, near))
    assert torch.equal(got, want)
    for a, b in zip(torch.autograd.grad(got, [far, w], d), torch.autograd.grad(want, [near, w], d)):
        assert torch.equal(a, b)
    q = mxfp4.quantize(w)
    got, want = mxfp4.linear(far, q), mxfp4.linear(near, q)
    assert torch.equal(got, want)
    dy = torch.empty_strided((B, V), (5 << 20, 1), dtype=torch.bfloat16, device=dev).copy_(want)  # cotangents as far apart
    assert torch.equal(torch.autograd.grad(got, far, dy)[0], torch.autograd.grad(want, near, dy.contiguous())[0])
    head = torch.empty_strided((V, H), (5 << 20, 1), dtype=torch.bfloat16, device=dev).copy_(w)
    assert torch.equal(linear_cross_entropy(near, head, t), linear_cross_entropy(near, w, t))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(2, 3, 5, 64), (2, 1, 15, 128), (3, 4, 45, 96)])
def test_linear_of_more_dimensions(dev, shape, dtype):
    """An input of four dimensions, dense or a view, has the bits of its rows, up to 64 of them and more."""
    import mxfp4
    g = torch.Generator(device=dev)
    g.manual_seed(shape[2])
    q = mxfp4.quantize(torch.randn(77, shape[-1], device=dev, generator=g))
    x = torch.randn(shape, device=dev, generator=g).to(dtype)
    rows = mxfp4.linear(x.reshape(-1, shape[-1]), q)
    assert torch.equal(mxfp4.linear(x, q).reshape(rows.shape), rows)
    assert torch.equal(mxfp4.linear(x.transpose(0, 2).contiguous().transpose(0, 2), q).reshape(rows.shape), rows)
    assert torch.equal(mxfp4.linear(lying(x.reshape(-1, shape[-1]), "off"), q), rows)
    assert torch.equal(mxfp4.linear(lying(x.reshape(-1, shape[-1]), "odd"), q), rows)
