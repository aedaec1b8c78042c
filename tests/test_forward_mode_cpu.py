"""Forward-mode tangents are refused where a kernel would leave them out (no kernel launches)."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import gdn_lib as L


def calls(x, w):
    """Calls of the operators with x [6, 64] and w [9, 64], and the tensors through which a tangent may come."""
    import mxfp4
    from embedding import embedding
    from linear_loss import linear_cross_entropy
    t = torch.zeros(6, dtype=torch.int64)
    q = mxfp4.Weight(torch.zeros(9, 32, dtype=torch.uint8), torch.zeros(9, 2, dtype=torch.uint8), 64)
    return {"linear_cross_entropy": lambda: linear_cross_entropy(x, w, t), "embedding": lambda: embedding(t, w),
            "linear": lambda: mxfp4.linear(x, q)}


@pytest.mark.parametrize("which", ["x", "w"])
def test_operators_at_both_ends(which):
    x, w = torch.randn(6, 64), torch.randn(9, 64)
    with fwAD.dual_level():
        dual = {"x": x, "w": w}
        dual[which] = fwAD.make_dual(dual[which], torch.ones_like(dual[which]))
        for name, call in calls(dual["x"], dual["w"]).items():
            takes = {"x": name != "embedding", "w": name != "linear"}[which]
            with pytest.raises(RuntimeError, match=f"{name} has no forward-mode" if takes else "ROCm GPU only"):
                call()
        for call in calls(x, w).values():  # an open level alone changes nothing
            with pytest.raises(RuntimeError, match="ROCm GPU only"):
                call()
    with pytest.raises(RuntimeError, match="linear_cross_entropy has no forward-mode"):
        torch.func.jvp(lambda a: calls(a, w)["linear_cross_entropy"](), (x,), (x,))


def test_backward_passes():
    """A cotangent with a tangent of its own would lose it in every backward pass."""
    g = torch.randn(3)
    with fwAD.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            L.once((g, fwAD.make_dual(g, g)), g)
        assert L.once((g, None), g)[0] is g or torch.equal(L.once((g, None), g)[0], g)


def test_operators_between():
    """The operators inside a model, each of its differentiable inputs in turn."""
    import grad_clip
    from gdn_engine import decode_step, recurrence
    from linear_attention import linear_attention, linear_attention_step
    from rotary import rotary, rotary_frequencies
    from token_logprobs import token_logprobs
    n = torch.randn
    inv, t, at = rotary_frequencies(4)[0], torch.zeros(2, 3, dtype=torch.int64), torch.arange(3)
    qkvg = [n(2, 3, 2, 8), n(2, 3, 2, 8), n(2, 3, 2, 8), -torch.rand(2, 3, 2), n(2, 2, 8, 8)]
    beta = torch.rand(2, 3, 2)
    for call, inputs in ((lambda q, k: rotary(q, k, at, inv), qkvg[:2]), (lambda z: token_logprobs(z, t), [n(2, 3, 9)]),
                         (lambda g: grad_clip.grad_norm([g]), [n(5)]), (lambda g: grad_clip.clip_grad_norm([g], 1.0), [n(5)]),
                         (linear_attention, qkvg),
                         (lambda q, k, v, g, s: recurrence(q, k, v, g, beta, s), qkvg),
                         (linear_attention_step, [*[a[:, 0] for a in qkvg[:4]], qkvg[4]]),
                         (lambda q, k, v, g, s: decode_step(q, k, v, g, beta[:, 0], s, s.detach().clone()),
                          [*[a[:, 0] for a in qkvg[:4]], qkvg[4]])):
        with pytest.raises(RuntimeError, match="ROCm GPU only"):
            call(*inputs)
        with fwAD.dual_level():
            for i in range(len(inputs)):
                with pytest.raises(RuntimeError, match="no forward-mode"):
                    call(*[fwAD.make_dual(a, torch.ones_like(a)) if i == j else a for j, a in enumerate(inputs)])
