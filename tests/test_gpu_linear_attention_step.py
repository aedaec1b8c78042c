"""GPU checks of linear attention's single tokens and autograd."""

import pytest
import torch

from test_gpu_linear_attention_decays import dev, inputs  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


def test_gradients_through_a_step_are_refused(dev):
    """A step's output and state depend on its inputs: a backward pass through either raises, instead of leaving them out."""
    from linear_attention import linear_attention, linear_attention_step
    q, k, v, g, state, dy, _ = inputs(dev, 2, 9, 1, 2, 64, 64, torch.float32, 5)
    g = g.expand(2, 9, 2)
    q.requires_grad_(True)
    S = state.clone()
    want = state.clone()
    with torch.no_grad():
        plain = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], want)
        assert not plain.requires_grad and not want.requires_grad
    y = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], S)
    assert torch.equal(y, plain) and torch.equal(S, want)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(y.sum(), q)
    y, _ = linear_attention(q[:, 1:], k[:, 1:], v[:, 1:], g[:, 1:], S)  # goes on from the state
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(y.sum(), q)
    y, _ = linear_attention(q[:, 1:], k[:, 1:], v[:, 1:], g[:, 1:], S.detach())
    assert bool(torch.autograd.grad(y.sum(), q)[0][:, 1:].any())
    for t in range(3):  # several steps; a part of a buffer of states, taken without gradients; a state that is a leaf
        linear_attention_step(q[:, t], k[:, t], v[:, t], g[:, t], S)
    with torch.no_grad():
        part = torch.stack([state, state])[1]
    leaf = state.clone().requires_grad_(True)
    for s in (part, leaf):
        y = linear_attention_step(q.detach()[:, 0] if s is leaf else q[:, 0], k[:, 0], v[:, 0], g[:, 0], s)
        assert torch.equal(y, plain) and torch.equal(s, want)
        with pytest.raises(RuntimeError, match="not differentiable"):
            torch.autograd.grad(y.sum(), leaf if s is leaf else q)
    y = linear_attention_step(q.detach()[:, 0], k[:, 0], v[:, 0], g[:, 0], state)
    assert not y.requires_grad and not state.requires_grad
