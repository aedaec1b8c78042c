"""GPU checks of the embedding lookup and its gradient against plain 64-bit forms.

A row of the lookup is a product in 64 bits, rounded to 32 and then to its type: half a step of each.  A gradient is a
64-bit sum of n terms in chunks of 32, at most n / 32 + 66 additions one after the other, each off by 2^-53 of a partial sum,
which sum |dy| bounds; then a product, and half a step of 32 bits and of its type.
"""

import math

import pytest
import torch

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


def plain(ids, w, dy, scale, padding):
    dev, ids, w, dy = w.device, ids.reshape(-1).cpu(), w.cpu(), dy.cpu()  # sums in order
    V = w.shape[0]
    ok = (ids >= 0) & (ids < V)
    y = torch.where(ok[:, None], w.double()[ids.clamp(0, V - 1)] * scale, math.nan)
    keep = ok if padding is None else ok & (ids != padding)
    rows, at = dy.reshape(len(ids), -1).double()[keep], ids[keep]
    dw = torch.zeros(w.shape, dtype=torch.float64, device=w.device).index_add_(0, at, rows) * scale
    size = torch.zeros(w.shape, dtype=torch.float64, device=w.device).index_add_(0, at, rows.abs()) * abs(scale)
    n = torch.zeros(V, dtype=torch.float64, device=w.device).index_add_(0, at, torch.ones_like(at, dtype=torch.float64))
    tol = size * ((n / 32 + 66) * 2.0 ** -53)[:, None] + (0 if w.dtype == torch.float32 else dw.abs() * U)
    return y.to(dev), dw.to(dev), tol.to(dev)


def within(got, want, tol, what):
    tol = tol + want.abs() * torch.finfo(got.dtype).eps / 2 + torch.finfo(got.dtype).smallest_normal
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    over = ((got.double() - want).abs() - tol)[torch.isfinite(want)]
    assert over.numel() == 0 or float(over.max()) <= 0, (what, float(over.max()))


def run(dev, ids, V, H, dtype, scale, padding, g):
    from embedding import embedding
    w = torch.randn(V, H, device=dev, generator=g).to(dtype).requires_grad_(True)
    dy = torch.randn(*ids.shape, H, device=dev, generator=g).to(dtype)
    y = embedding(ids, w, scale=scale, padding_idx=padding)
    assert y.shape == (*ids.shape, H) and y.dtype == dtype
    dw, = torch.autograd.grad(y, w, dy)
    wy, wdw, tol = plain(ids.long(), w.detach(), dy, scale, padding)
    within(y.detach().reshape(-1, H), wy, 0.0 if dtype == torch.float32 else wy.abs() * U, "y")
    within(dw, wdw, tol, "dw")
    return y, dw


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V,H", [(1, 1, 1), (1, 1000, 64), (7, 5, 70), (64, 300, 128), (1023, 50, 12), (1024, 50000, 8),
                                   (1025, 17, 33), (5000, 900, 257), (32768, 1000, 16), (32769, 3001, 24), (100000, 7, 8)])
def test_lookup_and_gradient(dev, N, V, H, dtype):
    print("embedding", N, V, H, dtype, flush=True)
    g = torch.Generator(device=dev)
    g.manual_seed(N + V)
    ids = (V ** torch.rand(N, device=dev, generator=g).double()).long().sub(1).clamp(0, V - 1)
    run(dev, ids, V, H, dtype, 1.0, None, g)
    run(dev, ids, V, H, dtype, -3.7, V // 2, g)


def test_a_million_tokens(dev):
    g = torch.Generator(device=dev)
    g.manual_seed(1)
    ids = torch.randint(0, 300, (3, 350001), device=dev, generator=g, dtype=torch.int32)
    ids[:, ::2] = 11
    run(dev, ids, 300, 8, torch.float32, 2.0, None, g)


@pytest.mark.parametrize("dtype", DTYPES)
def test_runs_against_chunks(dev, dtype):
    """Words whose tokens begin and end at every place of a chunk of 32, cover chunks exactly, and groups of 64 chunks."""
    g = torch.Generator(device=dev)
    g.manual_seed(2)
    for counts in (list(range(0, 70)), [32, 32, 64, 31, 1, 33, 63, 0, 96, 5], [2048, 2048, 4096, 2047, 1, 2049, 60000, 2048],
                   [31, 70000, 3], [70000], [65536 - 2048, 2048]):
        ids = torch.repeat_interleave(torch.arange(len(counts), device=dev), torch.tensor(counts, device=dev))
        ids = ids[torch.randperm(len(ids), device=dev, generator=g)]
        run(dev, ids, len(counts) + 1, 12, dtype, 1.5, None, g)
        run(dev, ids, len(counts), 12, dtype, 1.0, 0, g)


@pytest.mark.parametrize("dtype", DTYPES)
def test_ids_outside_and_padding(dev, dtype):
    """Ids outside the table give NaN rows; what their cotangents hold, or those of padding, reaches no gradient."""
    from embedding import embedding
    w = torch.randn(40, 64, device=dev).to(dtype).requires_grad_(True)
    ids = torch.tensor([3, -1, 40, 7, 7, -100, 1 << 40, 3, 9, -(1 << 62)], device=dev)
    dy = torch.randn(10, 64, device=dev).to(dtype)
    dy[[1, 2, 5, 6, 9]], dy[8] = math.nan, math.inf
    y = embedding(ids, w, padding_idx=9)
    dw, = torch.autograd.grad(y, w, dy)
    wy, wdw, tol = plain(ids, w.detach(), dy, 1.0, 9)
    within(y.detach(), wy, 0.0, "y")
    within(dw, wdw, tol, "dw")
    for only, n in ((torch.full((50,), 9, device=dev), 50), (ids[:0], 0)):  # nothing but padding, nothing at all
        y = embedding(only, w, padding_idx=9)
        assert y.shape == (n, 64)
        dw, = torch.autograd.grad(y, w, torch.ones_like(y))
        assert not dw.any()


def test_views(dev):
    """Tables and cotangents that are views; broadcast cotangents."""
    from embedding import embedding
    g = torch.Generator(device=dev)
    g.manual_seed(3)
    ids = torch.randint(0, 30, (4, 9), device=dev, generator=g)
    wide = torch.randn(30, 200, device=dev, generator=g)
    for w in (wide[:, 8:72], wide[:, 1:65], wide[:, ::2][:, :64], wide[::2][:15].repeat(2, 1)[:, 3:67], wide[:1, :64].expand(30, 64)):
        w = w.detach().requires_grad_(True)
        y = embedding(ids.t(), w, scale=2.0)
        big = torch.randn(9, 4, 100, device=dev, generator=g)
        for dy in (big[..., :64], big[..., 5:69], big.transpose(0, 1)[:, :, :64].transpose(0, 1), big[:1, :1, :64].expand(9, 4, 64),
                   torch.ones((), device=dev).expand(9, 4, 64)):
            dw, = torch.autograd.grad(y, w, dy, retain_graph=True)
            wy, wdw, tol = plain(ids.t(), w.detach(), dy, 2.0, None)
            within(dw, wdw, tol, "dw")
        within(y.detach().reshape(-1, 64), wy, 0.0, "y")


def test_module(dev):
    from embedding import Embedding
    torch.manual_seed(0)
    m = Embedding(50, 32, 4, scale=3.0)
    ids = torch.randint(0, 50, (3, 11))
    a = m(ids)
    a.sum().backward()
    ref = m.weight.grad.clone()
    m = m.to(dev)
    m.weight.grad = None
    b = m(ids.to(dev))
    b.sum().backward()
    assert torch.equal(a, b.cpu()) and torch.equal(m.weight.grad.cpu(), ref)
    assert torch.nn.Embedding(50, 32, 4).load_state_dict(m.state_dict())


def test_streams_and_graphs(dev):
    from embedding import embedding
    g = torch.Generator(device=dev)
    g.manual_seed(8)
    w = torch.randn(500, 128, device=dev, generator=g).bfloat16()
    ids = torch.randint(0, 500, (2000,), device=dev, generator=g)
    dy = torch.randn(2000, 128, device=dev, generator=g).bfloat16()

    def both():
        leaf = w.detach().requires_grad_(True)
        y = embedding(ids, leaf, scale=0.5, padding_idx=3)
        return [y.detach(), *torch.autograd.grad(y, leaf, dy)]

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
        ids.copy_(torch.randint(0, 500, (2000,), device=dev, generator=g))
        dy.copy_(torch.randn(2000, 128, device=dev, generator=g))
        want = both()
        for graph, out in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_second_gradients_are_refused(dev):
    from embedding import embedding
    w = torch.randn(5, 8, device=dev, requires_grad=True)
    dy = torch.randn(3, 8, device=dev, requires_grad=True)
    dw, = torch.autograd.grad(embedding(torch.arange(3, device=dev), w), w, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated twice"):
        torch.autograd.grad(dw.sum(), dy)
