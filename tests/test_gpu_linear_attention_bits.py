"""GPU checks of how many bits linear attention keeps of bf16 inputs: its outputs are as good as sums of 32 bits rounded once.

Tolerance, for every element: the output's own rounding, half a step (2^-8 of it), and what comes before, relative to the sum of
the terms' magnitudes (the same expression of the inputs' magnitudes): P and the state as operands in two terms (2^-17 each),
weights of fp32 exponentials (some 2^-23), fp32 sums of up to 200 terms with partial sums no larger than that (200 * 2^-24).
2^-15 is above all of them together.
"""

import pytest
import torch

from test_gpu_linear_attention import recurrence64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import gdn_lib
    gdn_lib.load()
    return torch.device("cuda:0")


# one token (a prompt's first, an output of one weight), a few, a chunk and its neighbours, several segments; every kernel:
# heads up to 64, 128 and 256 channels, in pairs and alone, sizes that are no multiple of 8
@pytest.mark.parametrize("size", [(2, 1, 1, 5, 64, 128), (1, 3, 2, 4, 128, 128), (3, 17, 1, 2, 64, 64), (2, 64, 1, 1, 128, 128),
                                  (1, 130, 2, 6, 96, 96), (1, 200, 1, 2, 256, 256), (1, 90, 1, 4, 80, 33), (1, 70, 1, 3, 33, 200),
                                  (1, 1100, 1, 2, 128, 64), (8, 600, 4, 8, 128, 128)])
@pytest.mark.parametrize("with_state", [False, True])
def test_bits_of_bf16(dev, size, with_state):
    from linear_attention import linear_attention
    print("bits", size, with_state, flush=True)
    B, T, Hk, Hv, Dk, Dv = size
    gen = torch.Generator(device=dev)
    gen.manual_seed(T)
    n = lambda *s: torch.randn(*s, device=dev, generator=gen)  # noqa: E731
    q, k, v, dy = n(B, T, Hk, Dk).bfloat16(), n(B, T, Hk, Dk).bfloat16(), n(B, T, Hv, Dv).bfloat16(), n(B, T, Hv, Dv).bfloat16()
    g = -torch.exp2(-torch.linspace(1.0, 8.0, Hv, device=dev)) * torch.nn.functional.softplus(n(B, T, Hv))
    state, dlast = n(B, Hv, Dv, Dk) if with_state else None, n(B, Hv, Dv, Dk)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    y, last = linear_attention(q, k, v, g, state)
    got = (y, *torch.autograd.grad([y, last], leaves, [dy, dlast]))
    want = recurrence64(q, k, v, g, state, Dk ** -0.5, dy, dlast)
    size = recurrence64(q.abs(), k.abs(), v.abs(), g, None if state is None else state.abs(), Dk ** -0.5, dy.abs(), dlast.abs())
    for x, i, name in zip(got, (0, 2, 3, 4), ("y", "dq", "dk", "dv")):
        room = want[i].abs() * 2.0 ** -8 + size[i] * 2.0 ** -15
        over = ((x.detach().double() - want[i]).abs() / room).max()
        print(name, f"{float(over):.3f}", flush=True)
        assert float(over) <= 1, (name, float(over))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("size", [(2, 1, 1, 5, 64, 128), (3, 17, 1, 2, 64, 64), (1, 130, 2, 6, 96, 96), (1, 200, 1, 2, 256, 256),
                                  (1, 90, 1, 4, 80, 33), (1, 1100, 1, 2, 128, 64)])
def test_bits_of_fp32_and_fp16(dev, size, dtype):
    """Every element, from states carried in: sums of less than 2^12 terms, whose errors of 2^-24 are independent (2^-18 of the
    terms' magnitudes; four times that), and in fp16 half a step of the output."""
    from linear_attention import linear_attention
    print("bits", size, dtype, flush=True)
    B, T, Hk, Hv, Dk, Dv = size
    gen = torch.Generator(device=dev)
    gen.manual_seed(T)
    n = lambda *s: torch.randn(*s, device=dev, generator=gen)  # noqa: E731
    q, k, v, dy = n(B, T, Hk, Dk).to(dtype), n(B, T, Hk, Dk).to(dtype), n(B, T, Hv, Dv).to(dtype), n(B, T, Hv, Dv).to(dtype)
    g = -torch.exp2(-torch.linspace(1.0, 8.0, Hv, device=dev)) * torch.nn.functional.softplus(n(B, T, Hv))
    state, dlast = n(B, Hv, Dv, Dk), n(B, Hv, Dv, Dk)
    leaves = [x.requires_grad_(True) for x in (q, k, v, state)]
    y, last = linear_attention(q, k, v, g, state)
    got = (y, last, *torch.autograd.grad([y, last], leaves, [dy, dlast]))
    want = recurrence64(q, k, v, g, state, Dk ** -0.5, dy, dlast)
    size = recurrence64(q.abs(), k.abs(), v.abs(), g, state.abs(), Dk ** -0.5, dy.abs(), dlast.abs())
    for x, i, name in zip(got, (0, 1, 2, 3, 4, 6), ("y", "last", "dq", "dk", "dv", "dstate")):
        room = size[i] * 2.0 ** -16 + (want[i].abs() * 2.0 ** -11 if x.dtype == torch.float16 else 0)
        over = float(((x.detach().double() - want[i]).abs() / room).max())
        print(name, f"{over:.3f}", flush=True)
        assert over <= 1, (name, over)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_heads_before_tokens(dev, dtype):
    """q, k, v and g as [B, H, T, D] transposed: the same bits as from contiguous copies, outputs and gradients."""
    from linear_attention import linear_attention
    B, T, Hk, Hv, Dk, Dv = 2, 150, 2, 4, 64, 40
    n = lambda *s: torch.randn(*s, device=dev)  # noqa: E731
    views = [n(B, Hk, T, Dk).to(dtype).transpose(1, 2), n(B, Hk, T, Dk).to(dtype).transpose(1, 2),
             n(B, Hv, T, Dv).to(dtype).transpose(1, 2), -torch.rand(B, Hv, T, device=dev).transpose(1, 2)]
    dy, out = n(B, T, Hv, Dv).to(dtype), []
    for leaves in (views, [x.contiguous() for x in views]):
        leaves = [x.detach().requires_grad_(True) for x in leaves]
        y, last = linear_attention(*leaves)
        out.append((y, last, *torch.autograd.grad([y, last], leaves, [dy, torch.ones_like(last)])))
    for a, b in zip(*out):
        assert torch.equal(a, b)
