"""GPU checks of the operators where a launch has more threads than fit in 32 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import gdn_lib
    gdn_lib.load()
    yield torch.device("cuda:0")
    torch.cuda.empty_cache()


def test_rotary_of_many_tokens(dev):
    """2^26 tokens and some, four to a workgroup of 256: each part of them as by itself."""
    from rotary import rotary
    T, part = (1 << 26) + 70001, 1 << 24
    q = torch.randn(1, T, 1, 2, device=dev).half()
    pos, inv = torch.arange(T, device=dev), torch.ones(1, device=dev, dtype=torch.float64)
    y, _ = rotary(q, q[:, :, :0], pos, inv)
    for t in range(0, T, part):
        want, _ = rotary(q[:, t:t + part], q[:, t:t + part, :0], pos[t:t + part], inv)
        assert torch.equal(y[:, t:t + part], want), t


def test_heads_added_over_many_elements(dev):
    """dq and dk of 2^24 tokens and some, 256 channels, of two value heads added in a launch of more than 2^32 threads.  Nothing
    but the last 2048 tokens has values or cotangents, so their gradients are those of these tokens alone: the same sums of fp32
    terms, cut into other segments (2^-16 of the whole, as in the other tests), and the rounding to fp16."""
    from linear_attention import linear_attention
    if torch.cuda.mem_get_info(dev)[0] < 100 << 30:
        pytest.skip("needs 100 GB of GPU memory")
    T, n = (1 << 24) + 64, 2048
    gen = torch.Generator(device=dev)
    gen.manual_seed(0)
    token = lambda: torch.randn(1, 1, 1, 256, device=dev, generator=gen).half()  # noqa: E731
    q, k, g = token(), token(), torch.tensor([-0.01, -0.1], device=dev)
    v, dy = (torch.zeros(1, T, 2, 1, device=dev, dtype=torch.float16) for _ in range(2))
    for x in (v, dy):
        x[:, -n:] = torch.randn(1, n, 2, 1, device=dev, generator=gen).half()

    def grads(T, v, dy):
        leaves = [x.expand(1, T, 1, 256).detach().requires_grad_(True) for x in (q, k)]
        return torch.autograd.grad(linear_attention(*leaves, v, g)[0], leaves, dy)

    want = [x.double() for x in grads(n, v[:, -n:], dy[:, -n:])]
    for got, w in zip(grads(T, v, dy), want):
        assert got.numel() > 1 << 32
        got = got[:, -n:].double()
        assert bool(torch.isfinite(got).all())
        assert float((got - w).norm() / w.norm()) <= 2 ** -16 + 2 ** -11


def test_step_of_many_sequences(dev):
    """More than 65535 heads over the batch.  States: one rounded product and sum (2^-23 of the terms); outputs sums of 16 of
    their products."""
    from linear_attention import linear_attention_step
    B, Hk, Hv, D = 2100, 2, 32, 16
    q, k = torch.randn(B, Hk, D, device=dev), torch.randn(B, Hk, D, device=dev)
    v, g, S = torch.randn(B, Hv, D, device=dev), -torch.rand(B, Hv, device=dev), torch.randn(B, Hv, D, D, device=dev)
    q64, k64 = (x.double().repeat_interleave(Hv // Hk, 1) for x in (q, k))
    old = S.double() * g.double().exp()[..., None, None]
    want, add = old + v.double()[..., None] * k64[..., None, :], v.double()[..., None] * k64[..., None, :]
    y = linear_attention_step(q, k, v, g, S)
    size = old.abs() + add.abs()
    assert bool(((S.double() - want).abs() <= 2.0 ** -21 * size).all())
    assert bool(((y.double() - 0.25 * (want * q64[..., None, :]).sum(-1)).abs()
                 <= 2.0 ** -20 * (size * q64[..., None, :].abs()).sum(-1)).all())
