"""GPU checks of MXFP4 weights and products with them against plain 64-bit forms.

Codes, scales and values are exact.  A product's sums are 32 bits over exact products (a bf16 weight value times at most three
bf16 terms of x): u = 2^-24, partial sums of K terms of size s within 4 sqrt(K) s, K independent roundings of them within 5
deviations are 20 u sum |x w|; then half a step of the result's type.
"""

import math

import pytest
import torch

import mxfp4_plain as P

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
U = 2.0 ** -24


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import gdn_lib
    gdn_lib.load()
    return torch.device("cuda:0")


def within(got, want, tol, what):
    tol = tol + want.abs() * torch.finfo(got.dtype).eps / 2 + torch.finfo(got.dtype).smallest_normal
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    over = ((got.double() - want).abs() - tol)[torch.isfinite(want)]
    assert over.numel() == 0 or float(over.max()) <= 0, (what, float(over.max()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,K", [(1, 1), (1, 32), (3, 33), (5, 64), (17, 100), (64, 2048), (33, 1001), (0, 64)])
def test_quantize(dev, N, K, dtype):
    import mxfp4
    g = torch.Generator(device=dev)
    g.manual_seed(N + K)
    w = torch.randn(N, K, device=dev, generator=g) * torch.exp2(20 * torch.rand(N, K, device=dev, generator=g).sub(0.5).round())
    w = w.to(dtype)
    w[torch.rand(N, K, device=dev, generator=g) < 0.1] = 0
    q = mxfp4.quantize(w)
    codes, scales = P.quantize(w)
    assert q.shape == (N, K) and torch.equal(q.scales, scales) and torch.equal(q.codes, codes)
    for out in DTYPES:
        got = mxfp4.dequantize(q, out)
        assert got.dtype == out and torch.equal(got, P.values(codes, scales, K).to(out))


def test_quantize_corners(dev):
    """Ties, the border of saturation, the smallest and largest numbers, zeros of either sign, infinite and NaN elements."""
    import mxfp4
    rows = torch.zeros(12, 64, device=dev)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 7.99, 4.0, 6.0, 0.2500001, 0.7499999, 1.2499999, 4.9999995])
    for i, e in enumerate((0, -130, -149, 100, 125)):
        rows[i, :15] = torch.ldexp(ties, torch.tensor(e)).to(dev)
        rows[i, 32:47] = -rows[i, :15]
    rows[5, :2] = torch.tensor([2.0 ** -149, -2.0 ** -149])
    rows[6, 0], rows[6, 40] = torch.finfo(torch.float32).max, -torch.finfo(torch.float32).max
    rows[7, 3], rows[8, 3], rows[9, 63] = math.inf, -math.inf, math.nan
    rows[10, ::2] = -0.0
    q = mxfp4.quantize(rows)
    codes, scales = P.quantize(rows)
    assert torch.equal(q.scales, scales) and torch.equal(q.codes, codes)
    want = P.values(codes, scales, 64)
    for out in DTYPES:
        assert torch.equal(mxfp4.dequantize(q, out).nan_to_num(7e4), want.to(out).nan_to_num(7e4))
    assert q.scales[7].tolist() == [255, 127 - 127] and q.scales[9, 1] == 255
    view = rows[:, 1:40]
    assert torch.equal(mxfp4.quantize(view).codes, P.quantize(view)[0])
    assert torch.equal(mxfp4.quantize(rows.t()).codes, P.quantize(rows.t())[0])


def make(dev, M, K, N, dtype, seed):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    import mxfp4
    w = K ** -0.5 * torch.randn(N, K, device=dev, generator=g) * torch.exp2(torch.randint(-6, 7, (N, 1), device=dev, generator=g))
    q = mxfp4.quantize(w)
    x = torch.randn(M, K, device=dev, generator=g).to(dtype)
    dy = torch.randn(M, N, device=dev, generator=g).to(dtype)
    return q, P.values(*q), x, dy


def check(x, dy, q, W):
    import mxfp4
    x = x.detach().requires_grad_(True)
    y = mxfp4.linear(x, q)
    assert y.shape == (*x.shape[:-1], W.shape[0]) and y.dtype == x.dtype
    X, D = x.detach().double(), dy.double()
    within(y.detach(), X @ W.t(), 20 * U * (X.abs() @ W.t().abs()), "y")
    dx, = torch.autograd.grad(y, x, dy)
    within(dx, D @ W, 20 * U * (D.abs() @ W.abs()), "dx")
    assert torch.equal(mxfp4.linear(x.detach(), q), y.detach())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (1, 2048, 100), (2, 32, 17), (16, 100, 33), (17, 1001, 64), (33, 256, 130),
                                   (64, 4096, 48), (65, 33, 40), (100, 128, 1), (130, 1001, 300), (257, 512, 1000),
                                   (1000, 250, 97), (700, 2048, 2048)])
def test_linear(dev, M, K, N, dtype):
    print("linear", M, K, N, dtype, flush=True)
    q, W, x, dy = make(dev, M, K, N, dtype, M + K + N)
    check(x, dy, q, W)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_pieces_of_the_weight(dev, dtype):
    """A copy of more than 2^26 elements."""
    q, W, x, dy = make(dev, 70, 2048, 33001, dtype, 5)
    check(x, dy, q, W)


@pytest.mark.parametrize("M", [3, 70])
def test_every_scale_and_code(dev, M):
    """One element of x is 1: rows of y are single values, at every scale and code (those that fp32 holds)."""
    import mxfp4
    scales = torch.arange(256, device=dev, dtype=torch.uint8)[:, None].expand(256, 2).contiguous()
    codes = (torch.arange(16, device=dev, dtype=torch.uint8) | torch.arange(16, device=dev, dtype=torch.uint8).flip(0) << 4)
    codes = codes.repeat(256, 2).contiguous()
    q = mxfp4.Weight(codes, scales, 64)
    want = P.values(*q)
    keep = (scales[:, 0] < 253)
    x = torch.zeros(M, 64, device=dev)
    for k in range(0, 64, 3):
        x.zero_()
        x[:, k] = 1
        for dtype in (torch.float32, torch.bfloat16):
            y = mxfp4.linear(x.to(dtype), q)
            assert torch.equal(y[:, keep], want[keep, k].to(dtype).expand(M, -1)), (k, dtype)
            assert torch.isnan(y[:, 255]).all()
    got = mxfp4.dequantize(q, torch.float32)
    assert torch.equal(got[keep], want[keep].float()) and torch.isnan(got[255]).all()


@pytest.mark.parametrize("M", [5, 90])
def test_views_and_odd_values(dev, M):
    """Strided, unaligned and transposed x and cotangents; NaN and infinite tokens, and the largest numbers, stay in their rows."""
    import mxfp4
    q, W, _, _ = make(dev, M, 96, 80, torch.float32, 3)
    g = torch.Generator(device=dev)
    g.manual_seed(4)
    for dtype in DTYPES:
        big = torch.randn(M, 300, device=dev, generator=g).to(dtype)
        for x, dy in ((big[:, :96], big[:, 100:180]), (big[:, 1:97], big[:, 3:83]), (big.t().contiguous().t()[:, :96], big[:, ::3][:, :80]),
                      (big[:1, :96].expand(M, 96), big[:1, :1].expand(M, 80))):
            check(x, dy, q, W)
        x = big[:, :96].contiguous()
        clean = mxfp4.linear(x, q)
        x[1, 5], x[2] = math.nan, math.inf
        y = mxfp4.linear(x, q)
        rest = [i for i in range(M) if i not in (1, 2)]
        assert torch.equal(y[rest], clean[rest]) and torch.isnan(y[1]).all()
        assert not torch.isfinite(y[2]).any()
    x = torch.full((M, 96), torch.finfo(torch.float32).max, device=dev)
    x[:, 1:] = 0
    assert torch.equal(mxfp4.linear(x, q), (W[:, :1].t() * x[:, :1].double()).float())
    wide = torch.randn(2, 3, M, 96, device=dev, generator=g)
    assert torch.equal(mxfp4.linear(wide, q), mxfp4.linear(wide.view(-1, 96), q).view(2, 3, M, 80)) or M == 5
    assert mxfp4.linear(wide[:0], q).shape == (0, 3, M, 80)


def test_streams_and_graphs(dev):
    import mxfp4
    for M in (9, 200):
        q, W, x, dy = make(dev, M, 256, 320, torch.bfloat16, 1)

        def both():
            leaf = x.detach().requires_grad_(True)
            y = mxfp4.linear(leaf, q)
            return [y.detach(), *torch.autograd.grad(y, leaf, dy), mxfp4.quantize(x).codes]

        want = both()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = both()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = both()
            graphs.append((graph, out))
        for _ in range(3):
            x.normal_()
            dy.normal_()
            want = both()
            for graph, out in graphs:
                graph.replay()
                torch.cuda.synchronize()
                assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_module(dev):
    import mxfp4
    torch.manual_seed(0)
    lin = torch.nn.Linear(96, 40, bias=False).to(dev)
    m = mxfp4.MXFP4Linear.of(lin)
    x = torch.randn(3, 7, 96, device=dev)
    assert torch.equal(m(x), mxfp4.linear(x, mxfp4.quantize(lin.weight)))
    other = mxfp4.MXFP4Linear.of(torch.nn.Linear(96, 40, bias=False).to(dev))
    other.load_state_dict(m.state_dict())
    assert torch.equal(other(x), m(x)) and not list(m.parameters())
    y = x.clone().requires_grad_(True)
    dy = torch.randn(3, 7, 40, device=dev, requires_grad=True)
    dx, = torch.autograd.grad(m(y), y, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated twice"):
        torch.autograd.grad(dx.sum(), dy)
