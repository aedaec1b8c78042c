"""GPU checks of linear attention against the recurrence in 64 bits, token by token, its gradients by the adjoint recurrence
and by differences.

Tolerances.  bf16 inputs: an output is a sum of two products whose inner operands (the pair weights, the state) are rounded
once more, half a step (2^-8) of an element at most; the rounding errors of a sum of many terms add up as independent ones,
so the relative error of a whole tensor (2-norms) is that of three roundings, below 3 * 2^-8 / sqrt(3) (a rounding's error is
spread evenly over half a step either way).  fp16 and fp32 inputs are fp32 inside: sums of some hundred terms of 2^-24 each,
2^-16 is far above their independent errors, and one rounding to fp16 (2^-11 / sqrt(3)) on top.  States are fp32 sums of
terms good to 2^-23 at least.
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


def recurrence64(q, k, v, g, state, scale, dy=None, dlast=None):
    """y, last and with dy the gradients (q, k, v, g per token, state), all float64."""
    q, k, v, g = (t.detach().double() for t in (q, k, v, g))
    B, T, Hk, Dk = q.shape
    Hv, Dv = v.shape[2:]
    r = Hv // Hk
    q, k = q.repeat_interleave(r, 2), k.repeat_interleave(r, 2)
    a = g.expand(B, T, Hv).exp()[..., None, None]
    S = torch.zeros(B, Hv, Dv, Dk, dtype=torch.float64, device=q.device) if state is None else state.detach().double()
    all_, ys = [S], []
    for t in range(T):
        S = a[:, t] * S + v[:, t, :, :, None] * k[:, t, :, None, :]
        all_.append(S)
        ys.append((S * q[:, t, :, None, :]).sum(-1) * scale)
    y = torch.stack(ys, 1)
    if dy is None:
        return y, S
    dy, D = dy.double(), dlast.double().clone()
    dq, dk, dv, dg = [torch.zeros_like(x) for x in (q, k, v)] + [torch.zeros(B, T, Hv, dtype=torch.float64, device=q.device)]
    for t in range(T - 1, -1, -1):
        dq[:, t] = scale * (all_[t + 1] * dy[:, t, :, :, None]).sum(-2)
        D = D + scale * dy[:, t, :, :, None] * q[:, t, :, None, :]
        dk[:, t] = (D * v[:, t, :, :, None]).sum(-2)
        dv[:, t] = (D * k[:, t, :, None, :]).sum(-1)
        dg[:, t] = (D * all_[t]).sum((-1, -2)) * a[:, t, :, 0, 0]
        D = a[:, t] * D
    fold = lambda x: x.unflatten(2, (Hk, r)).sum(3)  # noqa: E731
    return y, S, fold(dq), fold(dk), dv, dg, D


def near(got, want, rel, what):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, what
    assert bool(torch.isfinite(got).all()), what
    err = float((got - want).norm() / want.norm().clamp_min(1e-30))
    assert err <= rel, (what, err, rel)


def bounds(dtype):
    """(outputs of dtype, fp32 states)"""
    if dtype == torch.bfloat16:
        return 3 * 2 ** -8 / math.sqrt(3), 2 ** -16
    return 2 ** -16 + (2 ** -11 / math.sqrt(3) if dtype == torch.float16 else 0), 2 ** -16


def inputs(dev, B, T, Hk, Hv, Dk, Dv, dtype, per_head, with_state, seed):
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    n = lambda *s: torch.randn(*s, device=dev, generator=gen)  # noqa: E731
    q, k, v = n(B, T, Hk, Dk).to(dtype), n(B, T, Hk, Dk).to(dtype), n(B, T, Hv, Dv).to(dtype)
    rates = torch.exp2(-torch.linspace(1.0, 8.0, Hv, device=dev))
    g = -rates if per_head else -rates * torch.nn.functional.softplus(n(B, T, Hv))
    return q, k, v, g, n(B, Hv, Dv, Dk) if with_state else None, n(B, T, Hv, Dv).to(dtype), n(B, Hv, Dv, Dk)


def check(dev, B, T, Hk, Hv, Dk, Dv, dtype, per_head=False, with_state=True, seed=0, change=None):
    from linear_attention import linear_attention
    q, k, v, g, state, dy, dlast = inputs(dev, B, T, Hk, Hv, Dk, Dv, dtype, per_head, with_state, seed)
    if change is not None:
        q, k, v, g = change(q, k, v, g)
    leaves = [x.requires_grad_(True) for x in (q, k, v, g) + ((state,) if with_state else ())]
    y, last = linear_attention(q, k, v, g, state)
    grads = torch.autograd.grad([y, last], leaves, [dy, dlast])
    want = recurrence64(q, k, v, g, state, Dk ** -0.5, dy, dlast)
    out, st = bounds(dtype)
    assert y.dtype == dtype and last.dtype == torch.float32
    near(y, want[0], out, "y")
    near(last, want[1], st, "last")
    dg = want[5].sum((0, 1)) if per_head else want[5]
    for got, w, leaf, name in zip(grads, (*want[2:5], dg, want[6]), leaves, ("dq", "dk", "dv", "dg", "dstate")):
        assert got.dtype == leaf.dtype and got.shape == leaf.shape, name
        near(got, w, st if name == "dstate" else out, name)


SIZES = [  # one token, lengths around a chunk and a block, several segments; odd and unequal heads
    (1, 1, 1, 1, 128, 128), (2, 2, 1, 2, 64, 64), (1, 15, 2, 2, 32, 48), (2, 17, 1, 3, 80, 33), (1, 63, 1, 1, 128, 64),
    (1, 64, 2, 4, 128, 128), (3, 65, 1, 5, 64, 128), (1, 130, 3, 6, 96, 96), (1, 300, 1, 1, 256, 256),
    (1, 257, 1, 2, 200, 136), (2, 600, 2, 4, 128, 128), (1, 1031, 1, 2, 7, 5), (1, 900, 1, 1, 33, 256),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", SIZES)
def test_linear_attention(dev, size, dtype):
    print("linear attention", size, dtype, flush=True)
    B, T = size[:2]
    check(dev, *size, dtype, per_head=T % 2 == 0, with_state=B * T % 3 != 0, seed=T)


@pytest.mark.parametrize("dtype", DTYPES)
def test_views_of_one_projection(dev, dtype):
    """q, k and v as views of one buffer (an odd width too, so that rows are not aligned), g as a view."""
    from linear_attention import linear_attention
    gen = torch.Generator(device=dev)
    gen.manual_seed(1)
    for B, T, Hk, Hv, Dk, Dv, extra in ((2, 70, 2, 4, 64, 64, 0), (1, 131, 1, 2, 40, 33, 3), (2, 66, 1, 1, 128, 128, 1)):
        x = torch.randn(B, T, 2 * Hk * Dk + Hv * Dv + extra, device=dev, generator=gen).to(dtype)
        q, k = (x[..., i * Hk * Dk:(i + 1) * Hk * Dk].unflatten(-1, (Hk, Dk)) for i in (0, 1))
        v = x[..., 2 * Hk * Dk:2 * Hk * Dk + Hv * Dv].unflatten(-1, (Hv, Dv))
        g = -torch.rand(B, Hv, T, device=dev, generator=gen).transpose(1, 2)
        y, last = linear_attention(q, k, v, g)
        y2, last2 = linear_attention(q.contiguous(), k.contiguous(), v.contiguous(), g.contiguous())
        assert torch.equal(y, y2) and torch.equal(last, last2)
        want, S = recurrence64(q, k, v, g, None, Dk ** -0.5)
        near(y, want, bounds(dtype)[0], "y")
        near(last, S, bounds(dtype)[1], "last")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decays_at_their_ends(dev, dtype):
    """Decays of zero (log decay -inf) in the middle of a chunk, at its first and last token, and no decay at all."""
    def change(q, k, v, g):
        g = torch.zeros_like(g)
        for t in (0, 30, 63, 64, 127, 190):
            g[:, t] = -math.inf
        g[:, 100:110] = -20000.0
        g[:, 110:120] = -50.0
        return q, k, v, g
    check(dev, 2, 200, 1, 2, 64, 64, dtype, change=change)
    from linear_attention import linear_attention
    q, k, v, g, state, dy, dlast = inputs(dev, 1, 100, 1, 1, 64, 64, dtype, False, True, 5)
    g = torch.zeros_like(g).requires_grad_(True)
    with torch.no_grad():
        g[:, 50] = -math.inf
    y, last = linear_attention(q, k, v, g, state)
    y2, last2 = linear_attention(q[:, 50:], k[:, 50:], v[:, 50:], g[:, 50:].detach(), None)
    near(y[:, 50:], y2, 2 * bounds(dtype)[0], "restart")
    near(last, last2, bounds(dtype)[1], "restart")


def test_cotangents_one_at_a_time(dev):
    """A loss of y alone, of the final state alone; no gradient wanted for some inputs; broadcast cotangents."""
    from linear_attention import linear_attention
    q, k, v, g, state, dy, dlast = inputs(dev, 1, 90, 1, 2, 64, 64, torch.float32, False, True, 2)
    leaves = [x.requires_grad_(True) for x in (q, k, v, g, state)]
    for use_y, use_s in ((True, False), (False, True)):
        y, last = linear_attention(q, k, v, g, state)
        loss = (y.sum() if use_y else 0) + (last.sum() if use_s else 0)
        grads = torch.autograd.grad(loss, leaves)
        want = recurrence64(q, k, v, g, state, 0.125, torch.ones_like(dy) * use_y, torch.ones_like(dlast) * use_s)
        for a, b, n in zip(grads, want[2:], ("dq", "dk", "dv", "dg", "dstate")):
            if float(b.norm()):
                near(a, b, 2 ** -16, n)
            else:
                assert not bool(a.any()), n
    y, last = linear_attention(q, k.detach(), v, g.detach(), None)
    (dv,) = torch.autograd.grad(y.sum(), v)
    near(dv, recurrence64(q, k, v, g, None, 0.125, torch.ones_like(dy), torch.zeros_like(dlast))[4], 2 ** -16, "dv")


def test_gradients_by_differences(dev):
    """Along a random direction of every input, central differences of the fp32 forward."""
    from linear_attention import linear_attention
    q, k, v, g, state, dy, dlast = inputs(dev, 1, 150, 1, 2, 32, 48, torch.float32, True, True, 3)
    xs = [x.requires_grad_(True) for x in (q, k, v, g, state)]

    def loss(*a):
        y, last = linear_attention(*a)
        return (y.double() * dy.double()).sum() + (last.double() * dlast.double()).sum()

    grads = torch.autograd.grad(loss(*xs), xs)
    gen = torch.Generator(device=dev)
    gen.manual_seed(4)
    for i, gr in enumerate(grads):
        d = torch.randn(gr.shape, device=dev, generator=gen)
        d = d / d.norm() * xs[i].detach().norm()
        h = 2.0 ** -8
        with torch.no_grad():
            up, down = ([x + s * h * d if j == i else x for j, x in enumerate(xs)] for s in (1, -1))
            slope = float(loss(*up) - loss(*down)) / (2 * h)
            size = float(sum((t.double() ** 2).sum() for t in linear_attention(*xs))) ** 0.5
        # 2^-16 of outputs and cotangents of these sizes, over 2 h; the third derivative adds h^2
        room = 2 * 2 ** -16 * size * float((dy.norm() ** 2 + dlast.norm() ** 2) ** 0.5) / (2 * h)
        room += h * h * float(gr.double().norm() * d.double().norm())
        assert abs(slope - float((gr.double() * d.double()).sum())) <= room, i


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [(1, 1, 1, 128, 128), (3, 2, 4, 64, 64), (2, 1, 5, 80, 33), (5, 2, 2, 7, 5), (2, 1, 2, 256, 200)])
def test_step(dev, size, dtype):
    """Steps one after another against the recurrence and the whole sequence, with both kinds of decay."""
    from linear_attention import linear_attention, linear_attention_step
    print("step", size, dtype, flush=True)
    B, Hk, Hv, Dk, Dv = size
    for per_head in (False, True):
        q, k, v, g, state, _, _ = inputs(dev, B, 5, Hk, Hv, Dk, Dv, dtype, per_head, True, 6)
        S = state.clone()
        ys = [linear_attention_step(q[:, t], k[:, t], v[:, t], g if per_head else g[:, t], S) for t in range(5)]
        want, last = recurrence64(q, k, v, g, state, Dk ** -0.5)
        half = torch.finfo(dtype).eps / 2
        near(torch.stack(ys, 1), want, half + 2 ** -18, "y")
        near(S, last, 2 ** -20, "state")
        y, _ = linear_attention(q, k, v, g, state)
        near(y, want, bounds(dtype)[0], "whole")


def test_empty(dev):
    from linear_attention import linear_attention, linear_attention_step
    q, v = torch.zeros(2, 0, 1, 64, device=dev), torch.zeros(2, 0, 2, 32, device=dev)
    s = torch.randn(2, 2, 32, 64, device=dev, requires_grad=True)
    y, last = linear_attention(q, q, v, torch.zeros(2, 0, 2, device=dev), s)
    assert y.shape == (2, 0, 2, 32) and torch.equal(last, s)
    assert torch.equal(torch.autograd.grad(last.sum(), s)[0], torch.ones_like(s))
    y, last = linear_attention(q[:0], q[:0], v[:0], torch.zeros(2, device=dev))
    assert y.shape == (0, 0, 2, 32) and last.shape == (0, 2, 32, 64)
    z = torch.zeros(0, 1, 64, device=dev)
    assert linear_attention_step(z, z, z, torch.zeros(1, device=dev), torch.zeros(0, 1, 64, 64, device=dev)).shape == z.shape


def test_graph_and_other_stream(dev):
    """Forward, gradients and step captured once, replayed on new values, each replay equal to the eager call."""
    from linear_attention import linear_attention, linear_attention_step
    q, k, v, g, state, dy, dlast = inputs(dev, 1, 1100, 1, 2, 64, 64, torch.bfloat16, False, True, 8)
    S = state.clone()

    def work():
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v, g, state)]
        y, last = linear_attention(*leaves)
        grads = torch.autograd.grad([y, last], leaves, [dy, dlast])
        S.copy_(state)
        return (y.detach(), last.detach(), *grads, linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], S))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = work()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, work()):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
    for i in range(3):
        for t in (q, k, v, dy):
            t.copy_(torch.randn(t.shape, device=dev))
        state.copy_(torch.randn(state.shape, device=dev))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        for a, b in zip(got, work()):
            assert torch.equal(a, b), i


# four and six value heads on a key head (dq and dk of two heads added in one workgroup, the pairs afterwards), odd ratios
# (each head for itself), values too wide for two heads at a time; several segments
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [(1, 200, 1, 4, 128, 128), (2, 70, 2, 12, 64, 40), (1, 530, 1, 6, 64, 136), (1, 410, 1, 3, 256, 96),
                                  (1, 330, 1, 4, 255, 128)])
def test_heads_that_share_a_key_head(dev, size, dtype):
    print("linear attention", size, dtype, flush=True)
    check(dev, *size, dtype, per_head=size[3] == 12, seed=size[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_broadcast_inputs_and_far_apart_tokens(dev, dtype):
    """One key head expanded over three, one sequence's decays over the batch, a cotangent of one number; tokens 2^22 elements
    apart are copied.  The same bits twice: nothing depends on an order of arrival."""
    from linear_attention import linear_attention
    gen = torch.Generator(device=dev)
    gen.manual_seed(11)
    n = lambda *s: torch.randn(*s, device=dev, generator=gen)  # noqa: E731
    q, k, v = n(2, 150, 1, 64).to(dtype), n(2, 150, 1, 64).to(dtype), n(2, 150, 3, 32).to(dtype)
    g = -torch.rand(1, 150, 3, device=dev, generator=gen)
    leaves = [x.requires_grad_(True) for x in (q, k, v, g)]

    def run():
        y, last = linear_attention(q.expand(-1, -1, 3, -1), k.expand(-1, -1, 3, -1), v, g.expand(2, -1, -1))
        return y, last, torch.autograd.grad(y.float().sum(), leaves)

    y, last, grads = run()
    want = recurrence64(q, k, v, g, None, 0.125, torch.ones_like(y), torch.zeros_like(last))
    out, st = bounds(dtype)
    near(y, want[0], out, "y")
    near(last, want[1], st, "last")
    for got, w, name in zip(grads, (*want[2:5], want[5].sum(0, keepdim=True)), ("dq", "dk", "dv", "dg")):
        # torch adds the three heads' gradients in dtype: two more roundings
        near(got, w, out + 2 * torch.finfo(dtype).eps / 2, name)
    y2, last2, grads2 = run()
    assert torch.equal(y, y2) and torch.equal(last, last2) and all(map(torch.equal, grads, grads2))
    far = torch.zeros(3, 1 << 22, device=dev, dtype=dtype)
    far[:, :64] = q.detach()[0, :3, 0]
    x = far.as_strided((1, 3, 1, 64), (3 << 22, 1 << 22, 64, 1))
    with torch.no_grad():
        assert torch.equal(linear_attention(x, k[:1, :3], v[:1, :3], g[:, :3])[0],
                           linear_attention(q[:1, :3], k[:1, :3], v[:1, :3], g[:, :3])[0])


def test_stale_and_second_gradients_are_refused(dev):
    """A final state that a step has overwritten is not read by the backward pass, and gradients have none of their own."""
    from linear_attention import linear_attention, linear_attention_step
    q, k, v, g, state, dy, _ = inputs(dev, 1, 20, 1, 2, 64, 64, torch.float32, False, True, 12)
    q.requires_grad_(True)
    y, last = linear_attention(q, k, v, g, state)
    linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], last)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad((y * dy).sum(), q)
    y, _ = linear_attention(q, k, v, g, state)
    (dq,) = torch.autograd.grad((y * dy).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(dq.sum(), q)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes", [(2, 2, 4, 128, 128), (1, 1, 2, 64, 40), (1, 1, 1, 256, 33)])
def test_later_tokens_do_not_reach_earlier_outputs(dev, sizes, dtype):
    """Infinite and NaN values, keys, queries and decays of a token: outputs before it are those of the clean call, in its chunk
    too; sums may take another order (bounds)."""
    from linear_attention import linear_attention
    B, Hk, Hv, Dk, Dv = sizes
    for seed, t in enumerate((5, 37, 70, 199)):
        q, k, v, g, state, _, _ = inputs(dev, B, 200, Hk, Hv, Dk, Dv, dtype, False, True, 20 + seed)
        clean, _ = linear_attention(q, k, v, g, state)
        for what, bad in (("v", math.inf), ("v", math.nan), ("k", math.nan), ("q", math.inf), ("g", math.nan)):
            x = dict(q=q.clone(), k=k.clone(), v=v.clone(), g=g.clone())
            x[what][:, t, 0, ...] = bad
            y, last = linear_attention(x["q"], x["k"], x["v"], x["g"], state)
            near(y[:, :t], clean[:, :t], bounds(dtype)[0], (what, bad, t))
            assert not bool(torch.isfinite(y[:, t, 0]).any()), (what, bad, t)
            assert bool(torch.isfinite(last[:, 0]).all()) == (what == "q"), (what, bad, t)
    x = v.clone()
    x[:, 199, 0, 0] = math.nan  # one channel: the others are clean
    y, _ = linear_attention(q, k, x, g, state)
    near(y[..., 1:], clean[..., 1:], bounds(dtype)[0], "other channels")
    near(y[:, :199], clean[:, :199], bounds(dtype)[0], "earlier tokens")
    assert bool(y[:, 199, 0, 0].isnan().all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes", [(2, 2, 4, 128, 128), (1, 1, 3, 64, 40), (1, 1, 1, 256, 33)])
def test_nan_tokens_do_not_reach_gradients_they_have_no_part_in(dev, sizes, dtype):
    """A NaN key from which on nothing is in the loss: dq before it is the clean one.  A NaN query whose output is not in the
    loss: dk and dv after it are.  The same rounded operands, summed in another order: within the bounds."""
    from linear_attention import linear_attention
    B, Hk, Hv, Dk, Dv = sizes
    for seed, t in enumerate((5, 37, 70, 190)):
        q, k, v, g, state, dy, _ = inputs(dev, B, 200, Hk, Hv, Dk, Dv, dtype, False, True, 40 + seed)

        def grads(q, k, dy):
            leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
            return torch.autograd.grad(linear_attention(*leaves, g, state)[0], leaves, dy)

        bad, cut = k.clone(), dy.clone()
        bad[:, t, 0] = math.nan
        cut[:, t:] = 0
        near(grads(q, bad, cut)[0][:, :t], grads(q, k, cut)[0][:, :t], bounds(dtype)[0], ("dq", t))
        bad, cut = q.clone(), dy.clone()
        bad[:, t, 0] = math.nan
        cut[:, t] = 0
        for got, want, name in list(zip(grads(bad, k, cut), grads(q, k, cut), ("dq", "dk", "dv")))[1:]:
            near(got[:, t + 1:], want[:, t + 1:], bounds(dtype)[0], (name, t))
