"""GPU checks of rotary positions, token log probabilities and gradient clipping against plain 64-bit forms.

Tolerances count roundings: an output's own rounding is half a step of its type (eps / 2 relative), 32-bit arithmetic
before it a few times 2^-24 of the magnitudes that enter it (named where they are used).
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


def gen(dev, seed):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def within(got, want, tol, what):
    """|got - want| <= tol elementwise (all in 64 bits), equal where not finite."""
    got, want = got.double(), want.double()
    tol = torch.as_tensor(tol, dtype=torch.float64, device=want.device).expand_as(want)
    odd = ~torch.isfinite(want)
    assert got.shape == want.shape, what
    same = torch.where(torch.isnan(want), torch.isnan(got), got == want)
    assert bool(same[odd].all()), what
    over = ((got - want).abs() - tol)[~odd]
    assert over.numel() == 0 or float(over.max()) <= 0, (what, float(over.max()))


def half_step(t):
    return torch.finfo(t).eps / 2


# ------------------------------------------------------------------------------------------------ rotary


def rotary64(x, pos, inv, inter, factor, sign):
    x = x.double()
    R = 2 * inv.numel()
    a = (pos.double()[..., None] * inv.double()).reshape(-1, x.shape[1], 1, R // 2)
    c, s = a.cos() * factor, a.sin() * factor * sign
    p, q = (x[..., 0:R:2], x[..., 1:R:2]) if inter else (x[..., :R // 2], x[..., R // 2:R])
    y = x.clone()
    y[..., 0:R:2] if inter else None
    u, v = p * c - q * s, q * c + p * s
    size = (p * p + q * q).sqrt() * factor
    scale = x.abs()
    if inter:
        y[..., 0:R:2], y[..., 1:R:2] = u, v
        scale[..., 0:R:2], scale[..., 1:R:2] = size, size
    else:
        y[..., :R // 2], y[..., R // 2:R] = u, v
        scale[..., :R // 2], scale[..., R // 2:R] = size, size
    return y, scale


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,Hq,Hk,D,R", [(2, 5, 4, 2, 128, 128), (1, 1, 8, 8, 64, 32), (3, 7, 5, 1, 96, 24),
                                           (1, 2100, 2, 1, 80, 20), (2, 3, 1, 1, 7, 2), (2, 9, 3, 3, 256, 64),
                                           (1, 4, 2, 1, 2048, 1024)])
def test_rotary(dev, B, T, Hq, Hk, D, R, dtype, inter):
    from rotary import rotary, rotary_frequencies
    print("rotary", B, T, Hq, Hk, D, R, dtype, inter, flush=True)
    g = gen(dev, B * T + D)
    inv, factor = rotary_frequencies(R, scaling="parts", factor=4.0, device=dev)
    pos = torch.randint(0, 2_000_000, (B, T), device=dev, generator=g)
    q = torch.randn(B, T, Hq, D, device=dev, generator=g).to(dtype).requires_grad_(True)
    k = torch.randn(B, T, Hk, D, device=dev, generator=g).to(dtype).requires_grad_(True)
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    yq, yk = rotary(q, k, pos, inv, interleaved=inter, factor=factor)
    gq, gk = torch.autograd.grad([yq, yk], [q, k], [dq, dk])
    # two products, one sum, and sine and cosine of an angle rounded to 2^-25 turns: below 12 * 2^-24 of the pair's size
    for got, x, sign in ((yq, q, 1), (yk, k, 1), (gq, dq, -1), (gk, dk, -1)):
        want, size = rotary64(x.detach(), pos, inv, inter, factor, sign)
        assert got.dtype == dtype
        tiny = torch.finfo(dtype).smallest_normal
        within(got, want, want.abs() * half_step(dtype) + size * 12 * 2 ** -24 + tiny, "rotary")


def test_rotary_views_and_positions(dev):
    """q and k as views of one projection and as transposed heads, shared and 32-bit positions, one operand empty."""
    from rotary import rotary, rotary_frequencies
    g = gen(dev, 3)
    B, T, H, D = 2, 6, 3, 64
    inv, _ = rotary_frequencies(D, device=dev)
    x = torch.randn(B, T, 2 * H * D + 1, device=dev, generator=g)
    pos = torch.arange(100, 100 + T, device=dev, dtype=torch.int32)
    views = [(x[..., :H * D].unflatten(-1, (H, D)), x[..., H * D:-1].unflatten(-1, (H, D))),
             (x[..., 1:H * D + 1].unflatten(-1, (H, D)), x[..., H * D + 1:].unflatten(-1, (H, D))),
             (torch.randn(B, H, T, D, device=dev, generator=g).transpose(1, 2),
              torch.randn(B, T, D, H, device=dev, generator=g).transpose(2, 3))]
    for q, k in views:
        yq, yk = rotary(q, k, pos, inv.float())
        for got, src in ((yq, q), (yk, k)):
            want, size = rotary64(src, pos.expand(B, T), inv.float().double(), False, 1.0, 1)
            within(got, want, want.abs() * 2 ** -24 + size * 12 * 2 ** -24, "view")
    yq, yk = rotary(x[..., :H * D].unflatten(-1, (H, D)), x[..., :0].unflatten(-1, (0, D)), pos, inv)
    assert yk.shape == (B, T, 0, D) and yq.shape == (B, T, H, D)
    yq, _ = rotary(x[:, :0, :H * D].unflatten(-1, (H, D)), x[:, :0, :H * D].unflatten(-1, (H, D)), pos[:0], inv)
    assert yq.shape == (B, 0, H, D)


# ------------------------------------------------------------------------------------------------ log probabilities


def logprobs64(z, y, d, e, ignore=-100):
    z = z.detach().double()
    V = z.shape[-1]
    none = (z == -math.inf).all(-1)
    lp = torch.log_softmax(z, -1)
    lp = torch.where(none[:, None], torch.full_like(lp, -math.inf), lp)
    p = lp.exp()
    lp0 = torch.where(p > 0, lp, torch.zeros_like(lp))
    H = -(p * lp0).sum(-1)
    live = y != ignore
    logp = torch.where(live, lp.gather(1, y.clamp(0, V - 1)[:, None])[:, 0], torch.zeros_like(H))
    hot = torch.zeros_like(p)
    hot[torch.arange(len(y), device=y.device), y.clamp(0, V - 1)] = 1
    dd = (d.double() * live)[:, None]
    dz = dd * (hot - p) - e.double()[:, None] * p * (lp0 + H[:, None])
    dz = torch.where(none[:, None], torch.zeros_like(dz), dz)
    size = dd.abs() * (hot + p) + e.double().abs()[:, None] * p * (lp0.abs() + H[:, None])
    return logp, H, lp, dz, size


def check_logprobs(z, y, top, seed, targets_kept=True):
    from token_logprobs import token_logprobs
    dev = z.device
    g = gen(dev, seed)
    N, V = z.shape
    d, e = torch.randn(N, device=dev, generator=g), torch.randn(N, device=dev, generator=g)
    z = z.detach().requires_grad_(True)
    r = token_logprobs(z, y, entropy=True, top=top)
    (dz,) = torch.autograd.grad([r.logp, r.entropy], [z], [d, e])
    logp, H, lp, want_dz, size = logprobs64(z, y, d, e)
    # log s: every term of s is off by at most 2^-23 (1 + |x|), |x| < 90 where it counts; z - M and the two subtractions
    # round once each
    tol = 2 ** -23 * (1 + 90 / 8) + 2 ** -23 * z.detach().double().masked_fill(~(z.abs() < 1e30), 0).abs().amax(-1)
    within(r.logp, logp, tol + logp.masked_fill(~torch.isfinite(logp), 0).abs() * 2 ** -23, "logp")
    within(r.entropy, H, 4 * tol + H * 2 ** -22, "entropy")
    rel = 4 * tol[:, None] + 2 ** -23 * 100
    within(dz, want_dz, size * rel + want_dz.abs() * half_step(z.dtype) + torch.finfo(z.dtype).smallest_normal, "dlogits")
    if top:
        ids = torch.sort(z.detach().double(), dim=-1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(r.top_ids, ids)
        want = lp.gather(1, ids)
        within(r.top_logp, want, tol[:, None] + want.masked_fill(~torch.isfinite(want), 0).abs() * 2 ** -23, "top")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V,top", [(1, 1, 1), (3, 7, 7), (5, 1000, 5), (4, 8192, 64), (3, 8193, 20), (2, 40001, 32),
                                     (67, 513, 0), (1, 131072, 5)])
def test_logprobs(dev, N, V, top, dtype):
    print("logprobs", N, V, top, dtype, flush=True)
    g = gen(dev, N + V)
    z = (3 * torch.randn(N, V, device=dev, generator=g)).to(dtype)
    y = torch.randint(0, V, (N,), device=dev, generator=g)
    y[N // 2] = -100 if N > 1 else y[N // 2]
    check_logprobs(z, y, top, 1)


@pytest.mark.parametrize("V", [33, 20000])
def test_logprobs_ties_and_masks(dev, V):
    """Equal logits everywhere, signed zeros, one logit left, none left, masked alternatives, the type's lowest value."""
    g = gen(dev, V)
    z = torch.randn(8, V, device=dev, generator=g)
    z[0] = 1.5
    z[1] = 0.0
    z[1, ::3] = -0.0
    z[2] = -math.inf
    z[2, V - 2] = 4.0
    z[3] = -math.inf
    z[4, 2:] = -math.inf
    z[5] = torch.finfo(torch.float32).min
    z[5, 7] = 1.0
    z[6] = (z[6] * 2).round()
    y = torch.tensor([0, V - 1, V - 2, 3, 1, 7, 5, -100], device=dev)
    check_logprobs(z, y, 20, 2)
    check_logprobs(z.bfloat16(), y, 20, 2)


def test_logprobs_nan_inf_and_bad_targets(dev):
    from token_logprobs import token_logprobs
    z = torch.randn(4, 300, device=dev).requires_grad_(True)
    with torch.no_grad():
        z[0, 5] = math.nan
        z[1, 7] = math.inf
    y = torch.tensor([1, 2, 300, -1], device=dev)
    r = token_logprobs(z, y, entropy=True, top=2)
    assert bool(torch.isnan(r.logp).all())
    assert bool(torch.isnan(r.entropy[:2]).all()) and bool(torch.isfinite(r.entropy[2:]).all())
    assert int(r.top_ids[0, 0]) == 5 and int(r.top_ids[1, 0]) == 7
    (dz,) = torch.autograd.grad(r.logp.sum(), z)
    assert bool(torch.isnan(dz).all(-1).all())


def test_logprobs_shifted_view_and_single_outputs(dev):
    """logits[:, :-1] is read in place; a loss of logp alone, of entropy alone, of neither."""
    from token_logprobs import token_logprobs
    g = gen(dev, 5)
    z = torch.randn(3, 9, 1001, device=dev, generator=g).requires_grad_(True)
    y = torch.randint(0, 1001, (3, 8), device=dev, generator=g)
    w = torch.randn(3, 8, device=dev, generator=g)
    zero = torch.zeros(24, device=dev)
    flat = z.detach()[:, :-1].reshape(-1, 1001)
    for pick in ("logp", "entropy"):
        r = token_logprobs(z[:, :-1], y, entropy=True)
        (dz,) = torch.autograd.grad((getattr(r, pick) * w).sum(), z)
        d, e = (w.flatten(), zero) if pick == "logp" else (zero, w.flatten())
        want = logprobs64(flat, y.flatten(), d, e)[3].view(3, 8, 1001)
        within(dz[:, :-1], want, 1e-5 * w.abs()[..., None].double(), pick)
        assert not bool(dz[:, -1].any())
    strided = token_logprobs(z.detach().transpose(0, 2).contiguous().transpose(0, 2)[:, :-1], y)
    assert torch.equal(strided.logp, token_logprobs(z.detach()[:, :-1], y).logp)
    assert token_logprobs(z[:, :0], y[:, :0]).logp.shape == (3, 0)


# ------------------------------------------------------------------------------------------------ clipping


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("limit", [0.5, 1e9])
def test_clip(dev, norm_type, limit):
    """Mixed types and sizes (more tensors than one launch holds, empty and single ones, odd addresses, transposed and
    strided views), in place and into other tensors."""
    from grad_clip import clip_grad_norm, grad_norm
    print("clip", norm_type, limit, flush=True)
    g = gen(dev, 9)
    base = torch.randn(70001, device=dev, generator=g)
    ts = [base[1:5000], base[5001:5002], base[6000:6000], base[10000:70000].view(300, 200).t()]
    wide = torch.randn(40, 50, device=dev, generator=g)
    ts.append(wide[:, 3:40])
    for i in range(260):
        n = 1 + 37 * i
        ts.append(torch.randn(n, device=dev, generator=g).to(DTYPES[i % 3]))
    ts.append(torch.randn(3, 100000, device=dev, generator=g).bfloat16())
    before = [t.double().clone() for t in ts]
    flat = torch.cat([b.flatten() for b in before])
    want = flat.norm() if norm_type == 2.0 else flat.abs().max()
    factor = min(1.0, limit / (float(want) + 1e-6))
    outs = [torch.empty_like(t, memory_format=torch.contiguous_format) for t in ts]
    norms = [grad_norm(ts, norm_type), clip_grad_norm(ts, limit, norm_type, out=outs),
             clip_grad_norm(ts, limit, norm_type)]
    for n in norms:
        assert n.dtype == torch.float32 and n.shape == ()
        within(n, want, want.abs() * 2 ** -24, "norm")
    for t, o, b in zip(ts, outs, before):
        w = b * factor  # the factor and the product round once each, then the type
        tol = w.abs() * (half_step(t.dtype) + 2 ** -22) + torch.finfo(t.dtype).smallest_normal
        within(t, w, tol, "in place")
        within(o, w, tol, "out")
    assert float(wide[0, 0].double()) != 0 and torch.equal(torch.cat([t.flatten().double() for t in outs]),
                                                            torch.cat([t.flatten().double() for t in ts]))


def test_clip_far_values_and_odd_ones(dev):
    from grad_clip import clip_grad_norm, grad_norm
    big = torch.full((5000,), 1e30, device=dev)
    within(grad_norm([big]), torch.tensor(1e30 * math.sqrt(5000.0), device=dev, dtype=torch.float64),
           1e30 * math.sqrt(5000.0) * 2 ** -23, "squares past 32 bits")
    small = torch.full((5000,), 1e-30, device=dev)
    within(grad_norm([small]), torch.tensor(float(small[0]) * math.sqrt(5000.0), device=dev, dtype=torch.float64),
           1e-28 * 2 ** -22, "squares below 32 bits")
    a = torch.ones(10, device=dev)
    a[3] = math.inf
    n = clip_grad_norm([a], 1.0)
    assert float(n) == math.inf and bool(torch.isnan(a[3])) and float(a[0]) == 0.0
    for t in (2.0, math.inf):
        b, c = torch.ones(3000, device=dev), torch.ones(2, device=dev)
        b[2999] = math.nan
        assert math.isnan(float(clip_grad_norm([b, c], 1.0, t))) and bool(torch.isnan(c).all())
    z = torch.zeros(7, device=dev)
    assert float(clip_grad_norm([z], 0.0)) == 0.0 and not bool(z.any())
    with pytest.raises(ValueError, match="share memory"):
        clip_grad_norm([a, a], 1.0)
    with pytest.raises(ValueError, match="share memory"):
        clip_grad_norm([a[:6], a[5:]], 1.0)
    with pytest.raises(ValueError, match="share memory"):
        clip_grad_norm([a[:4], a[4:8]], 1.0, out=[a[4:8], a[:4]])


def test_operators_in_a_graph_and_on_another_stream(dev):
    """Captured once, replayed on new values, each replay equal to the eager call."""
    from grad_clip import clip_grad_norm
    from rotary import rotary, rotary_frequencies
    from token_logprobs import token_logprobs
    inv, _ = rotary_frequencies(64, device=dev)
    q, k = torch.randn(2, 3, 4, 64, device=dev), torch.randn(2, 3, 2, 64, device=dev)
    pos = torch.arange(3, device=dev)
    z, y = torch.randn(6, 9000, device=dev), torch.randint(0, 9000, (6,), device=dev)
    gs = [torch.randn(5000, device=dev), torch.randn(33, device=dev).bfloat16()]
    outs = [torch.empty_like(x) for x in gs]

    def work():
        r = token_logprobs(z, y, entropy=True, top=4)
        return (*rotary(q, k, pos, inv), r.logp, r.entropy, r.top_ids, r.top_logp, clip_grad_norm(gs, 1.0, out=outs),
                *outs)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
    for i in range(3):
        for t in (q, k, z, *gs):
            t.copy_(torch.randn(t.shape, device=dev) * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        for a, b in zip(got, work()):
            assert torch.equal(a, b), i


def test_second_gradients_and_overwritten_tensors_are_refused(dev):
    from grad_clip import clip_grad_norm
    from rotary import rotary, rotary_frequencies
    from token_logprobs import token_logprobs
    z = torch.randn(3, 50, device=dev, requires_grad=True)
    (dz,) = torch.autograd.grad(token_logprobs(z, torch.arange(3, device=dev)).logp.sum(), z, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(dz.sum(), z)
    q, w = (torch.randn(1, 4, 2, 8, device=dev, requires_grad=True) for _ in range(2))
    inv, _ = rotary_frequencies(8)
    a, _ = rotary(q, q.detach(), torch.arange(4, device=dev), inv.to(dev))
    (dq,) = torch.autograd.grad((a * w).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(dq.sum(), w)
    x = torch.randn(10, device=dev, requires_grad=True)
    p = x.exp()  # its gradient reads p
    clip_grad_norm([p.detach()], 1e-3)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(p.sum(), x)
