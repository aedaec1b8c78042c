"""GPU checks of the cross entropy of x W^T without logits, against a plain 64-bit form.

Tolerances count roundings, u = 2^-24.  A logit is a 32-bit sum of exact products of 16-bit inputs: partial sums of H terms of
size s stay within 4 sqrt(H) s, and H independent roundings of them within 5 deviations are 20 u sum |x w|; fp32 inputs are two
fp16 terms, whose products miss 3 * 2^-22 |x w| more.  A probability is off by the relative error of e^(z - lse): twice the
logits' error and a few u; stored as a 16-bit difference it loses 2^-11 of itself (fp32 inputs: 2^-22, as the other operand).
The smallest step of an fp16 number is 2^-24.  Differences are stored times 2^15: half a step is 2^-40 (fp32 inputs, the second
term times 2^11 more: 2^-51), for the weight's gradient relative to the power of two above the largest cotangent.  The other
operand is stored with its largest magnitude below 2^15: half a step is 2^-39 of it at most.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import gdn_lib
    gdn_lib.load()
    return torch.device("cuda:0")


def inputs(dev, N, H, V, dtype, seed, ignored=True):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    x = torch.randn(N, H, device=dev, generator=g).to(dtype)
    w = (3 * H ** -0.5 * torch.randn(V, H, device=dev, generator=g)).to(dtype)
    t = torch.randint(0, V, (N,), device=dev, generator=g)
    if ignored and N > 2:
        t[torch.rand(N, device=dev, generator=g) < 0.3] = -100
    return x, w, t, torch.randn(N, device=dev, generator=g)


def plain(x, w, t, d, ignore=-100):
    """(loss, dx, dw) in 64 bits and their tolerances before the results' own rounding."""
    wide = x.dtype == torch.float32
    live = t != ignore
    X = torch.where(live[:, None], x.detach().double(), 0.0)
    W = w.detach().double()
    V = W.shape[0]
    z = X @ W.t()
    zerr = ((20 * U + (3 * 2.0 ** -22 if wide else 0)) * (X.abs() @ W.abs().t())).amax(1)
    lse = torch.logsumexp(z, 1)
    at = t.clamp(0, V - 1)[:, None]
    bad = live & ((t < 0) | (t >= V))
    loss = torch.where(live, lse - z.gather(1, at)[:, 0], 0.0)
    loss[bad] = math.nan
    loss_tol = 2 * zerr + U * (16 + 4 * loss.abs().nan_to_num() + 4 * z.abs().amax(1))
    D = torch.where(live, d.double(), 0.0)
    D[bad] = math.nan
    p = (z - lse[:, None]).exp()
    diff = p.clone()
    diff[torch.arange(len(t), device=t.device), at[:, 0]] -= 1
    rel = (2.0 ** -22 * 3 if wide else 2.0 ** -11) + 20 * U
    # the difference's own error: relative to itself as stored, relative to p as computed
    derr = diff.abs() * rel + p * (2 * zerr[:, None] + 40 * U)
    floor, A = 2.0 ** -51 if wide else 2.0 ** -40, D.abs()
    dx = D[:, None] * (diff @ W)
    dx_tol = A[:, None] * ((derr + floor) @ W.abs() + diff.abs().sum(1, keepdim=True) * 2.0 ** -39 * W.abs().max())
    dw = (D[:, None] * diff).t() @ X
    most = 2 * A.nan_to_num().max()
    dw_tol = (A[:, None] * derr + most * floor * live[:, None]).t() @ X.abs()
    dw_tol += (A[:, None] * diff.abs()).sum(0)[:, None] * 2.0 ** -39 * X.nan_to_num(0, 0, 0).abs().max()
    return (loss, dx, dw), (loss_tol, dx_tol, dw_tol)


def within(got, want, tol, what):
    tol = tol + want.abs() * torch.finfo(got.dtype).eps / 2 + torch.finfo(got.dtype).smallest_normal
    got = got.double()
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    over = ((got - want).abs() - tol)[~odd]
    assert over.numel() == 0 or float(over.max()) <= 0, (what, float(over.max()))


DTYPES = [torch.bfloat16, torch.float16, torch.float32]
SIZES = [(1, 64, 100), (5, 70, 130), (3, 1, 2), (33, 256, 1000), (64, 128, 129), (100, 64, 1), (200, 128, 3001),
         (300, 1001, 777), (515, 2048, 5000), (2, 192, 50001)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,H,V", SIZES)
def test_loss_and_gradients(dev, N, H, V, dtype):
    from linear_loss import linear_cross_entropy
    print("loss", N, H, V, dtype, flush=True)
    x, w, t, d = inputs(dev, N, H, V, dtype, N + H + V)
    x.requires_grad_(True)
    w.requires_grad_(True)
    want, tol = plain(x, w, t, d)
    loss = linear_cross_entropy(x, w, t, reduction="none")
    assert loss.dtype == torch.float32 and loss.shape == t.shape
    within(loss.detach(), want[0], tol[0], "loss")
    dx, dw = torch.autograd.grad(loss, [x, w], d)
    assert dx.dtype == dtype and dw.dtype == dtype
    within(dx, want[1], tol[1], "dx")
    within(dw, want[2], tol[2], "dw")
    assert not dx[t == -100].any() and not loss[t == -100].any()
    only = linear_cross_entropy(x.detach(), w.detach(), t, reduction="none")
    assert torch.equal(only, loss.detach())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,H,V", [(2100, 320, 66001), (500, 64, 140001)])
def test_several_pieces(dev, N, H, V, dtype):
    """More than 2^26 differences, the last piece short; each gradient alone."""
    from linear_loss import linear_cross_entropy
    print("pieces", N, H, V, dtype, flush=True)
    x, w, t, d = inputs(dev, N, H, V, dtype, 7)
    want, tol = plain(x, w, t, d)
    x.requires_grad_(True)
    loss = linear_cross_entropy(x, w, t, reduction="none")
    dx, = torch.autograd.grad(loss, [x], d)
    within(loss.detach(), want[0], tol[0], "loss")
    within(dx, want[1], tol[1], "dx")
    x = x.detach()
    w.requires_grad_(True)
    dw, = torch.autograd.grad(linear_cross_entropy(x, w, t, reduction="none"), [w], d)
    within(dw, want[2], tol[2], "dw")


@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_reductions(dev, reduction):
    from linear_loss import linear_cross_entropy
    x, w, t, _ = inputs(dev, 70, 128, 500, torch.float32, 11)
    x, t = x.view(2, 35, 128).requires_grad_(True), t.view(2, 35)
    w.requires_grad_(True)
    n = int((t != -100).sum()) if reduction == "mean" else 1
    loss = linear_cross_entropy(x, w, t, reduction=reduction)
    assert loss.shape == ()
    got = torch.autograd.grad(2 * loss, [x, w])
    want, tol = plain(x.view(70, 128), w, t.view(-1), torch.full((70,), 2.0 / n, device=dev))
    total = want[0].sum() / n
    assert abs(float(loss) - float(total)) <= float(tol[0].sum()) / n + U * abs(float(total))
    within(got[0].view(70, 128), want[1], tol[1] + want[1].abs() * 4 * U, "dx")
    within(got[1], want[2], tol[2] + want[2].abs() * 4 * U, "dw")


def test_nothing_counts(dev):
    from linear_loss import linear_cross_entropy
    x = torch.full((6, 64), math.nan, device=dev, dtype=torch.bfloat16, requires_grad=True)
    w = torch.randn(50, 64, device=dev, dtype=torch.bfloat16, requires_grad=True)
    for t, ignore in ((torch.full((6,), -100, device=dev), -100), (torch.full((6,), 3, device=dev, dtype=torch.int32), 3)):
        loss = linear_cross_entropy(x, w, t, ignore_index=ignore)
        assert float(loss) == 0
        dx, dw = torch.autograd.grad(loss, [x, w])
        assert not dx.any() and not dw.any()
    empty = linear_cross_entropy(x[:0], w, t[:0])
    assert float(empty) == 0
    dx, dw = torch.autograd.grad(empty, [x, w])
    assert not dx.any() and not dw.any()
    assert linear_cross_entropy(x[:0], w, t[:0], reduction="none").shape == (0,)


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_places_hold_anything(dev, dtype):
    """Infinite, NaN and huge inputs at ignored tokens reach nothing; a bad target and a NaN token reach what they enter."""
    from linear_loss import linear_cross_entropy
    x, w, t, d = inputs(dev, 90, 128, 400, dtype, 5, ignored=False)
    t[:8] = -100
    big = torch.finfo(dtype).max
    x[0], x[1], x[2, 3], x[3] = math.nan, math.inf, -math.inf, big
    x.requires_grad_(True)
    w.requires_grad_(True)
    want, tol = plain(x, w, t, d)
    loss = linear_cross_entropy(x, w, t, reduction="none")
    dx, dw = torch.autograd.grad(loss, [x, w], d)
    for g, a, b in zip((loss.detach(), dx, dw), want, tol):
        within(g, a, b, "masked")
    t[20], t[21] = 400, -1
    loss = linear_cross_entropy(x, w, t, reduction="none")
    dx, dw = torch.autograd.grad(loss, [x, w], d)
    want, tol = plain(x, w, t, d)
    within(loss.detach(), want[0], tol[0], "bad target")
    within(dx, want[1], tol[1], "bad target")
    assert torch.isnan(dw).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("share", [0.0, 0.3, 0.97, 1.0])
@pytest.mark.parametrize("N,H,V", [(2048, 64, 300), (2111, 200, 1501)])
def test_tokens_left_out(dev, N, H, V, share, dtype):
    """Long batches, of which products see only the tokens that count: none left out, some, nearly all, all."""
    from linear_loss import linear_cross_entropy
    print("left out", N, H, V, share, dtype, flush=True)
    x, w, t, d = inputs(dev, N, H, V, dtype, int(100 * share) + N, ignored=False)
    out = torch.rand(N, device=dev) < share
    t[out] = 7
    x[out] = math.nan
    x.requires_grad_(True)
    w.requires_grad_(True)
    want, tol = plain(x, w, t, d, 7)
    loss = linear_cross_entropy(x, w, t, ignore_index=7, reduction="none")
    dx, dw = torch.autograd.grad(loss, [x, w], d)
    for got, a, b, what in zip((loss.detach(), dx, dw), want, tol, ("loss", "dx", "dw")):
        within(got, a, b, what)
    assert not dx[t == 7].any() and not loss[t == 7].any()
    mean = linear_cross_entropy(x, w, t, ignore_index=7)
    n = int((t != 7).sum())
    assert abs(float(mean.detach()) - float(want[0].sum()) / max(1, n)) <= float(tol[0].sum()) / max(1, n) + U * abs(float(mean))
    if share == 0.3:  # a target that is no word
        t[(t != 7).nonzero()[3]] = V
        x = x.detach().requires_grad_(True)
        want, tol = plain(x, w, t, d, 7)
        loss = linear_cross_entropy(x, w, t, ignore_index=7, reduction="none")
        dx, = torch.autograd.grad(loss, [x], d)
        within(loss.detach(), want[0], tol[0], "loss")
        within(dx, want[1], tol[1], "dx")


def test_views_and_magnitudes(dev):
    """Strided rows, unaligned bases, and inputs whose size fp16 does not hold."""
    from linear_loss import linear_cross_entropy
    g = torch.Generator(device=dev)
    g.manual_seed(2)
    for dtype in (torch.bfloat16, torch.float32):
        wide = torch.randn(40, 3 * 128 + 1, device=dev, generator=g).to(dtype)
        head = torch.randn(300, 2 * 128, device=dev, generator=g).to(dtype) * 0.2
        t = torch.randint(0, 300, (40,), device=dev, generator=g)
        d = torch.randn(40, device=dev, generator=g)
        for x, w in ((wide[:, 128:256], head[:, 128:]), (wide[:, 1:129], head[:, :128]),
                     (wide[:, :128].t().contiguous().t(), head[:, ::2]), (wide[:, :128] * 2.0 ** -70, head[:, :128] * 2.0 ** 60),
                     (wide[:, :128] * 2.0 ** 40, head[:, :128] * 2.0 ** -50)):
            x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
            want, tol = plain(x, w, t, d)
            loss = linear_cross_entropy(x, w, t, reduction="none")
            dx, dw = torch.autograd.grad(loss, [x, w], d)
            for a, b, c in zip((loss.detach(), dx, dw), want, tol):
                within(a, b, c, "view")


def test_difference_quotients(dev):
    """The gradients against the loss itself, moved by 2^-9 along random directions (error of the quotient: the loss's over
    2^-8, and a sixth of the third derivative, below 2^-18)."""
    from linear_loss import linear_cross_entropy
    x, w, t, _ = inputs(dev, 24, 96, 200, torch.float32, 3)
    g = torch.Generator(device=dev)
    g.manual_seed(4)
    X, W = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    grads = torch.autograd.grad(linear_cross_entropy(X, W, t), [X, W])
    for i, (a, grad) in enumerate(zip((x, w), grads)):
        v = torch.randn(a.shape, device=dev, generator=g)
        v /= v.norm()
        e = 2.0 ** -9
        up, down = [linear_cross_entropy(*((a + s * e * v, w) if i == 0 else (x, a + s * e * v)), t).double() for s in (1, -1)]
        assert abs(float((up - down) / (2 * e)) - float((grad.double() * v).sum())) <= 2.0 ** -11


def test_streams_graphs_and_repeats(dev):
    """Another stream than the tensors' own, and captured graphs replayed among eager calls, give the eager bits."""
    from linear_loss import linear_cross_entropy
    for N in (130, 2300):
        streams_graphs_and_repeats(dev, N, linear_cross_entropy)


def streams_graphs_and_repeats(dev, N, linear_cross_entropy):
    x, w, t, _ = inputs(dev, N, 128, 700, torch.bfloat16, 9)

    def both(x, w, t):
        x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        loss = linear_cross_entropy(x, w, t)
        return [loss.detach(), *torch.autograd.grad(loss, [x, w])]

    want = both(x, w, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both(x, w, t)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got
    graphs = []
    xs = x.clone()
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = both(xs, w, t)
        graphs.append((graph, out))
    for seed in range(3):
        x2, _, t2, _ = inputs(dev, N, 128, 700, torch.bfloat16, 20 + seed)
        t.copy_(t2)  # others are left out
        want = both(x2, w, t)
        xs.copy_(x2)
        for graph, out in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_second_gradients_are_refused(dev):
    from linear_loss import linear_cross_entropy
    x, w, t, _ = inputs(dev, 8, 64, 50, torch.float32, 1)
    x.requires_grad_(True)
    dx, = torch.autograd.grad(linear_cross_entropy(x, w, t), [x], create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated twice"):
        torch.autograd.grad(dx.sum(), [x])
    y = x.detach().clone().requires_grad_(True)
    leaf = y * 1
    loss = linear_cross_entropy(leaf, w, t)
    with torch.no_grad():
        leaf.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()


@pytest.mark.parametrize("N,H,V", [(1, 64, 1), (1, 2048, 5000), (17, 192, 129), (33, 320, 3001), (64, 64, 128), (65, 1024, 777),
                                   (128, 512, 4099), (129, 64, 300)])
def test_few_fp32_scores(dev, N, H, V):
    """Without gradients, few tokens, fp32 weights read as they lie (up to 128 tokens): three terms of each number are exact, and
    the products left out, of a second and a third term, are below 2 * 2^-22 of the factors' product."""
    from linear_loss import linear_cross_entropy
    print("scores", N, H, V, flush=True)
    x, w, t, _ = inputs(dev, N, H, V, torch.float32, 11)
    if N > 2:
        t[2] = -100
        x[2] = math.nan  # of a token that does not count
    want, tol = plain(x, w, t, torch.zeros(N, device=dev))
    within(linear_cross_entropy(x, w, t, reduction="none"), want[0], tol[0], "loss")
    rows = torch.full((V, H + 4), math.nan, device=dev)[:, :H].copy_(w)  # rows apart, still aligned
    within(linear_cross_entropy(x, rows, t, reduction="none"), want[0], tol[0], "rows apart")
    odd = torch.full((V * H + 1,), math.nan, device=dev)[1:].view(V, H).copy_(w)  # not aligned
    within(linear_cross_entropy(x, odd, t, reduction="none"), want[0], tol[0], "not aligned")


def test_few_fp32_scores_of_odd_values(dev):
    """Magnitudes that no scale of fp16 terms would span, infinite words, NaN and targets that are no word."""
    from linear_loss import linear_cross_entropy
    N, H, V = 20, 128, 500
    x, w, t, _ = inputs(dev, N, H, V, torch.float32, 12, ignored=False)
    x[:, 0] *= 2.0 ** -60
    w[:, 0] *= 2.0 ** 60
    x[:, 1] *= 2.0 ** 50
    w[:, 1] *= 2.0 ** -50
    t[3], t[4] = V, -7
    want, tol = plain(x, w, t, torch.zeros(N, device=dev))
    within(linear_cross_entropy(x, w, t, reduction="none"), want[0], tol[0], "loss")
    t[3] = t[4] = 0
    for odd in (-math.inf, math.nan, math.inf):  # no number of terms adds up to an infinity: it counts as NaN
        w[9, 5] = odd
        assert bool(torch.isnan(linear_cross_entropy(x, w, t, reduction="none")).all())


@pytest.mark.parametrize("V,dtype", [(1_060_001, torch.bfloat16), (530_001, torch.float32)])
def test_weights_beyond_32_bits(dev, V, dtype):
    """A weight of more than 2^32 bytes, targets at both of its ends."""
    from linear_loss import linear_cross_entropy
    N, H = 8, 2048
    print("large weight", V, dtype, flush=True)
    x, w, t, d = inputs(dev, N, H, V, dtype, 13, ignored=False)
    t[0], t[1], t[2] = V - 1, 0, -100
    want, tol = plain(x, w, t, d)
    x.requires_grad_(True)
    w.requires_grad_(True)
    loss = linear_cross_entropy(x, w, t, reduction="none")
    dx, dw = torch.autograd.grad(loss, [x, w], d)
    within(loss.detach(), want[0], tol[0], "loss")
    within(dx, want[1], tol[1], "dx")
    for rows in (slice(0, 2000), slice(V // 2, V // 2 + 2000), slice(V - 2000, V)):
        within(dw[rows], want[2][rows], tol[2][rows], "dw")
