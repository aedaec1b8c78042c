"""GPU checks of the decays' gradients of linear attention: every head for itself, against the recurrence in 64 bits.

dg_t = a_t <dS_t, S_{t-1}> is the sum of what crosses t: the pairs of its chunk, a_r = q_r . dq_r and b_s = k_s . dk_s of the
parts that come through the state, and c, which a chain of a's and b's carries from chunk to chunk between products of the
states themselves.

Tolerances, of one head's gradients as a whole (2-norms), so that no head hides behind another.  e is the error of an a or a b
relative to the norms that enter it: for bf16 inputs the state goes into them in two terms of 8 bits (2^-16 at most), for fp32
and fp16 inputs they are fp32 sums of up to 128 terms (2^-24 each, independent: 2^-20 is far above).  The products of the states
are at most 8 chunks apart and the chain runs from the nearer end, so c carries the errors of at most 4 * 64 a's and as many b's,
independent ones: with memories of tau tokens, e sqrt(512 / tau) of a c, below 8 e for memories from 8 tokens on (shorter ones
hold nothing at a chunk's end).  8 * 2^-16 = 2^-13 per token, 2^-17 in fp32; twice that, as half a step is not the error's only
source.  One decay for a head adds up its tokens: within 8 chunks the error of c is one number for all of them, while the
gradients themselves add up as tau-long stretches: another factor sqrt(512 / tau) < 8.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import gdn_lib
    gdn_lib.load()
    return torch.device("cuda:0")


def tolerance(dtype):
    """(per token, per head)"""
    t = 2.0 ** -12 if dtype == torch.bfloat16 else 2.0 ** -16
    return t, 8 * t


def states64(q, k, v, g, state, scale, dy, dlast=None):
    """dL/dg of every token [B, T, Hv] = a_t <dS_t, S_{t-1}>, float64, from the states of all tokens (sums of q . dq - k . dk,
    which need no states, lose what has faded)."""
    q, k, v, g, dy = (t.detach().double() for t in (q, k, v, g, dy))
    B, T, Hk, Dk = q.shape
    Hv = v.shape[2]
    q, k = (x.repeat_interleave(Hv // Hk, 2) for x in (q, k))
    a = g.expand(B, T, Hv).exp()[..., None, None]
    S = [q.new_zeros(B, Hv, v.shape[-1], Dk) if state is None else state.detach().double()]
    for t in range(T):
        S.append(a[:, t] * S[-1] + v[:, t, :, :, None] * k[:, t, :, None, :])
    D = torch.zeros_like(S[0]) if dlast is None else dlast.double()
    out = q.new_empty(B, T, Hv)
    for t in range(T - 1, -1, -1):
        D = D + scale * dy[:, t, :, :, None] * q[:, t, :, None, :]
        out[:, t] = (D * S[t]).sum((-1, -2)) * a[:, t, :, 0, 0]
        D = a[:, t] * D
    return out


def each_head(got, want, rel, what):
    """2-norms over everything but the last axis."""
    got, want = got.detach().double().flatten(0, -2), want.flatten(0, -2)
    assert bool(torch.isfinite(got).all()), what
    err = (got - want).norm(dim=0) / want.norm(dim=0).clamp_min(1e-30)
    print(what, f"{float(err.max()):.3g} of {rel:.3g}", flush=True)
    assert float(err.max()) <= rel, (what, err.tolist(), rel)


def inputs(dev, B, T, Hk, Hv, Dk, Dv, dtype, seed):
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    n = lambda *s: torch.randn(*s, device=dev, generator=gen)  # noqa: E731
    q, k, v = n(B, T, Hk, Dk).to(dtype), n(B, T, Hk, Dk).to(dtype), n(B, T, Hv, Dv).to(dtype)
    g = -torch.exp2(-torch.linspace(0.0, 12.0, Hv, device=dev))  # memories of one token to thousands
    return q, k, v, g, n(B, Hv, Dv, Dk), n(B, T, Hv, Dv).to(dtype), n(B, Hv, Dv, Dk)


def gradient(q, k, v, g, state, dy, dlast=None):
    from linear_attention import linear_attention
    g = g.detach().clone().requires_grad_(True)
    y, last = linear_attention(q, k, v, g, state)
    outs, cots = ([y], [dy]) if dlast is None else ([y, last], [dy, dlast])
    return torch.autograd.grad(outs, g, cots)[0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,t0", [(64, 40), (61, 16), (33, 32), (64, 5)])
def test_large_pairs_after_a_token_leave_its_gradient_alone(dev, T, t0, dtype):
    """Values and queries 2^10 times larger from t0 on: the pairs among those tokens are 2^20 times the size of the others, and
    dg before t0 holds none of them."""
    q, k, v, g, _, dy, _ = inputs(dev, 2, T, 1, 3, 64, 64, dtype, T + t0)
    late = torch.arange(T, device=dev) >= t0
    v = torch.where(late[:, None, None], v * 2 ** 10, v)
    k = torch.where(late[:, None, None], k * 2 ** 10, k)
    g = g.expand(2, T, 3) * torch.rand(2, T, 3, device=dev)
    dg = gradient(q, k, v, g, None, dy)
    want = states64(q, k, v, g, None, 0.125, dy)
    each_head(dg[:, 1:t0], want[:, 1:t0], tolerance(dtype)[0], f"dg before {t0} of {T}, {dtype}")
    each_head(dg, want, tolerance(dtype)[0], f"dg of {T}, {dtype}")


# as many sequences and heads as fill the card without cutting the sequence, and few heads, whose sequence is cut
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,Hk,Hv,D", [(16, 6001, 2, 32, 32), (2, 6001, 2, 16, 64)])
def test_long_sequences(dev, B, T, Hk, Hv, D, dtype):
    """A decay for every token, then the same decays one for each head: the errors of many chunks do not add up.  Per head: of
    the sequences' sums."""
    q, k, v, g, state, dy, dlast = inputs(dev, B, T, Hk, Hv, D, D, dtype, B)
    want = states64(q, k, v, g, state, D ** -0.5, dy, dlast)
    per_token, per_head = tolerance(dtype)
    each_head(gradient(q, k, v, g.expand(B, T, Hv), state, dy, dlast), want, per_token, f"dg of {B} x {T}, {dtype}")
    got = gradient(q, k, v, g, state, dy, dlast).double()
    size = want.sum(1).norm(dim=0)  # of the B sums that a head's gradient adds
    err = (got - want.sum((0, 1))).abs() / size
    print(f"per head {float(err.max()):.3g}", flush=True)
    assert float(err.max()) <= per_head, err.tolist()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,Hk,Hv,D", [(16, 4100, 2, 32, 32), (1, 4100, 1, 8, 64)])
def test_loss_of_the_last_tokens(dev, B, T, Hk, Hv, D, dtype):
    """Nothing but the last ten outputs in the loss: what they draw from thousands of tokens earlier fades, and so does the
    error.  Per token, every 512 tokens for themselves where the gradient is above 2^-40 of the last one."""
    q, k, v, g, state, dy, _ = inputs(dev, B, T, Hk, Hv, D, D, dtype, 7)
    dy[:, :-10] = 0
    want = states64(q, k, v, g, state, D ** -0.5, dy)
    got = gradient(q, k, v, g.expand(B, T, Hv), state, dy).double()
    per_token, per_head = tolerance(dtype)
    each_head(got, want, per_token, f"dg of the last tokens, {B} x {T}, {dtype}")
    size = want.norm(dim=(0, 1))
    for t in range(0, T, 512):
        part, err = want[:, t:t + 512].norm(dim=(0, 1)), (got - want)[:, t:t + 512].norm(dim=(0, 1))
        on = part > 2.0 ** -40 * size
        assert bool((err[on] <= per_token * part[on]).all()), (t, (err / part).tolist())
    err = (gradient(q, k, v, g, state, dy).double() - want.sum((0, 1))).abs() / want.sum(1).norm(dim=0)
    print(f"per head {float(err.max()):.3g}", flush=True)
    assert float(err.max()) <= per_head, err.tolist()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes", [(2, 2, 4, 128, 128), (1, 1, 3, 64, 40), (1, 1, 1, 256, 33), (40, 1, 16, 32, 32)])
def test_odd_tokens_do_not_reach_decays_they_have_no_part_in(dev, sizes, dtype):
    """A NaN or infinite value or key of token t is in no state before t: dg up to t is the clean one.  A NaN or infinite query or
    cotangent of token t is in no cotangent of a state after t: dg from t + 1 on is.  Both with and without the final state in
    the loss, in sequences of several chunks and of several segments (few heads) or one (many)."""
    B, Hk, Hv, Dk, Dv = sizes
    T = 1300
    q, k, v, g, state, dy, dlast = inputs(dev, B, T, Hk, Hv, Dk, Dv, dtype, 3)
    g = g.expand(B, T, Hv) * (0.5 + torch.rand(B, T, Hv, device=dev))
    for with_last in (True, False):
        end = dlast if with_last else None
        clean = gradient(q, k, v, g, state, dy, end).double()
        for t in (0, 5, 63, 64, 700, 1151, 1299):
            for what, bad in (("v", math.nan), ("v", math.inf), ("k", math.nan), ("q", math.nan), ("dy", math.nan),
                              ("dy", -math.inf)):
                x = dict(q=q.clone(), k=k.clone(), v=v.clone(), dy=dy.clone())
                x[what][:, t, 0] = bad
                dg = gradient(x["q"], x["k"], x["v"], g, state, x["dy"], end)
                part = slice(0, t + 1) if what in ("v", "k") else slice(t + 1, T)
                if clean[:, part].numel():
                    # two results, each within its tolerance of the exact ones
                    each_head(dg[:, part], clean[:, part], 2 * tolerance(dtype)[0], (what, bad, t, with_last))
                each_head(dg[..., Hv // Hk:], clean[..., Hv // Hk:], 2 * tolerance(dtype)[0], "other heads") if Hk > 1 else None


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_nan_where_no_loss_is_left(dev, dtype):
    """A NaN key from which on nothing is in the loss: the gradients of the decays up to it are the clean ones."""
    q, k, v, g, state, dy, _ = inputs(dev, 1, 900, 1, 2, 64, 64, dtype, 4)
    g = g.expand(1, 900, 2)
    for t in (30, 64, 511, 899):
        cut = dy.clone()
        cut[:, t:] = 0
        bad = k.clone()
        bad[:, t] = math.nan
        each_head(gradient(q, bad, v, g, state, cut)[:, :t + 1], gradient(q, k, v, g, state, cut)[:, :t + 1].double(),
                  2 * tolerance(dtype)[0], t)


def test_one_decay_for_a_head_in_32_bits(dev):
    """fp32: products of the states at most four chunks apart, two chunks of a's and b's from the nearer end.  As in the head of
    this file, with e = 2^-22 (sums of 128 terms, 2^-24 each, independent) and 256 in the place of 512: e * 256 / tau of the
    size of a head's sums, for the three longest of these memories (tau = 64 to 256) 2^-20.  Over eight sequences, one by one."""
    B, T, Hv, D = 8, 2047, 3, 128
    q, k, v, _, state, dy, dlast = inputs(dev, B, T, 1, Hv, D, D, torch.float32, 9)
    g = -torch.exp2(-torch.tensor([6.0, 7.0, 8.0], device=dev))
    want = states64(q, k, v, g, state, D ** -0.5, dy, dlast).sum(1)
    got = torch.stack([gradient(q[b:b + 1], k[b:b + 1], v[b:b + 1], g, state[b:b + 1], dy[b:b + 1], dlast[b:b + 1])
                       for b in range(B)]).double()
    err = (got - want).norm(dim=0) / want.norm(dim=0)
    print("one decay for a head", err.tolist(), flush=True)
    assert float(err.max()) <= 2.0 ** -20, err.tolist()
