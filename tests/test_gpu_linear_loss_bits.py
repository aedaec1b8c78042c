"""GPU checks of how many bits the gradients of the cross entropy without logits keep: those of 16-bit inputs are as good as sums
of 32 bits rounded once, and small probabilities keep theirs.

Tolerances count roundings, u = 2^-24, as in test_gpu_linear_loss.py.  bf16: a difference is two bf16 terms, each off by half a
step of what it rounds, so by 2^-16 of itself; x, the head and the powers of two are exact.
"""

import pytest
import torch

from test_gpu_linear_loss import U, dev, within  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


def case(dev, N, H, V, seed, apart):
    """Tokens and words in bf16; every third word's logits lie ``apart`` below the others'."""
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    x = torch.randn(N, H, device=dev, generator=g)
    w = 2 * H ** -0.5 * torch.randn(V, H, device=dev, generator=g)
    x[:, 0] = 1
    w[:, 0] = 0
    w[2::3, 0] = -apart
    t = torch.randint(0, (V + 1) // 3, (N,), device=dev, generator=g) * 3
    if N > 2:
        t[torch.rand(N, device=dev, generator=g) < 0.2] = -100
    return x.bfloat16(), w.bfloat16(), t, torch.randn(N, device=dev, generator=g)


def exact(x, w, t, d):
    """dx and dW in 64 bits, the bounds of what comes before their own rounding, and the probabilities."""
    X, W, D = x.double(), w.double(), torch.where(t != -100, d.double(), 0.0)
    z = X @ W.t()
    p = (z - torch.logsumexp(z, 1, keepdim=True)).exp()
    zerr = (20 * U * (X.abs() @ W.abs().t())).amax(1, keepdim=True)
    diff = p.clone()
    diff[torch.arange(len(t), device=t.device), t.clamp_min(0)] -= 1
    err = D.abs()[:, None] * (diff.abs() * (2.0 ** -16 + 20 * U) + p * (2 * zerr + 40 * U + 2 * U * z.abs()))
    diff = D[:, None] * diff
    return (diff @ W, diff.t().contiguous() @ X), (err @ W.abs(), err.t().contiguous() @ X.abs()), p


SIZES = [(1, 64, 7), (130, 64, 9), (300, 128, 300), (600, 64, 12), (700, 200, 501), (2100, 96, 11), (2500, 256, 1300)]


def gradients(x, w, t, d, wanted):
    from linear_loss import linear_cross_entropy
    leaves = [a.detach().requires_grad_(n in wanted) for n, a in (("x", x), ("w", w))]
    loss = linear_cross_entropy(*leaves, t, reduction="none")
    return torch.autograd.grad(loss, [a for a in leaves if a.requires_grad], d)


@pytest.mark.parametrize("N,H,V", SIZES)
def test_bits_of_bf16_gradients(dev, N, H, V):
    """Every element; and as far from 64 bits as the exact gradients rounded once, up to a difference of 2^-16 beneath a rounding
    of some 2^-9.6 (root of the mean square, of the whole): 2^-13.8 of it.  1 / 500 leaves room for both."""
    print("bits", N, H, V, flush=True)
    x, w, t, d = case(dev, N, H, V, N + V, 0.0)
    want, tol, _ = exact(x, w, t, d)
    for wanted in ("xw", "x", "w"):
        got = gradients(x, w, t, d, wanted)
        for g, a, b, what in zip(got, *zip(*[(want[i], tol[i], "d" + n) for i, n in enumerate("xw") if n in wanted])):
            within(g, a, b, what)
            if a.numel() >= 1 << 13:
                far, least = float((g.double() - a).norm()), float((a.bfloat16().double() - a).norm())
                print(what, wanted, f"{far / least:.5f}", flush=True)
                assert far <= least * (1 + 1 / 500), (what, wanted, far / least)


@pytest.mark.parametrize("N,H,V", SIZES)
@pytest.mark.parametrize("apart", [24.0, 48.0, 64.0])
def test_bits_of_small_probabilities(dev, N, H, V, apart):
    """Words of probabilities down to 2^-110, whose second term is still a normal number, have gradients of their own size."""
    print("small", N, H, V, apart, flush=True)
    x, w, t, d = case(dev, N, H, V, N + V, apart)
    want, tol, p = exact(x, w, t, d)
    rows = (p > 2.0 ** -110).all(0)
    assert bool(rows[2]) or apart > 48
    for wanted in ("xw", "w"):
        dw = gradients(x, w, t, d, wanted)[-1]
        within(dw[rows], want[1][rows], tol[1][rows], "dw")
        assert bool(dw[rows].any(1).all())


@pytest.mark.parametrize("N,H,V", [(1, 64, 7), (20, 128, 500), (33, 70, 129), (64, 192, 1000), (128, 64, 3001)])
def test_few_fp32_tokens_of_any_magnitude(dev, N, H, V):
    """Channels whose factors lie up to 2^120 apart, of up to 128 tokens with fp32 words: loss and gradients of one channel do not
    suffer from another's magnitude.  Three terms hold every number; the products that are left out, of a second and a third term,
    are below 2 * 2^-22 of the factors' product (3 here)."""
    from linear_loss import linear_cross_entropy
    print("magnitudes", N, H, V, flush=True)
    g = torch.Generator(device=dev)
    g.manual_seed(N + V)
    x = torch.randn(N, H, device=dev, generator=g)
    w = 3 * H ** -0.5 * torch.randn(V, H, device=dev, generator=g)
    for c, e in ((0, 60), (1, -50), (2, 20), (H - 1, -33)):
        x[:, c] *= 2.0 ** -e
        w[:, c] *= 2.0 ** e
    t = torch.randint(0, V, (N,), device=dev, generator=g)
    if N > 2:
        t[1] = -100
    d = torch.randn(N, device=dev, generator=g)
    X, W, D = x.double(), w.double(), torch.where(t != -100, d.double(), 0.0)
    z = X @ W.t()
    lse = torch.logsumexp(z, 1, keepdim=True)
    p = (z - lse).exp()
    at = (torch.arange(N, device=dev), t.clamp_min(0))
    loss = torch.where(t != -100, lse[:, 0] - z[at], 0.0)
    part = 20 * U + 3 * 2.0 ** -22  # of a product of two sums of terms, and of sums of them
    zerr = part * (X.abs() @ W.abs().t()).amax(1, keepdim=True)
    diff = p.clone()
    diff[at] -= 1
    err = D.abs()[:, None] * (diff.abs() * part + p * (2 * zerr + 40 * U + 2 * U * z.abs().amax(1, keepdim=True)))
    diff = D[:, None] * diff
    x.requires_grad_(True)
    w.requires_grad_(True)
    got = linear_cross_entropy(x, w, t, reduction="none")
    dx, dw = torch.autograd.grad(got, [x, w], d)
    within(got.detach(), loss, 2 * zerr[:, 0] + U * (16 + 4 * loss.abs() + 4 * z.abs().amax(1)), "loss")
    within(dx, diff @ W, err @ W.abs(), "dx")
    within(dw, diff.t().contiguous() @ X, err.t().contiguous() @ X.abs(), "dw")


@pytest.mark.parametrize("N,H,V", [(129, 64, 300), (200, 70, 1501), (2111, 192, 777)])
def test_fp32_tokens_leave_others_alone(dev, N, H, V):
    """A huge token and a tiny one among others: each token's loss and dx are as good as its own numbers allow."""
    from linear_loss import linear_cross_entropy
    from test_gpu_linear_loss import inputs, plain
    print("huge token", N, H, V, flush=True)
    x, w, t, d = inputs(dev, N, H, V, torch.float32, N)
    t[5] = t[9] = 3
    x[5] *= 2.0 ** 40
    x[9] *= 2.0 ** -50
    x.requires_grad_(True)
    want, tol = plain(x, w, t, d)
    loss = linear_cross_entropy(x, w, t, reduction="none")
    dx, = torch.autograd.grad(loss, [x], d)
    within(loss.detach(), want[0], tol[0], "loss")
    within(dx, want[1], tol[1], "dx")
    within(linear_cross_entropy(x.detach(), w, t, reduction="none"), want[0], tol[0], "loss alone")
