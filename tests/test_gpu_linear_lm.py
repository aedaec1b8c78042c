"""GPU checks of the example language model: the operators together in a training step and in decoding."""

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


def test_decoding_token_by_token_equals_the_whole_sequence(dev):
    """The states of a prompt carried through single tokens give the logits of the whole sequence.  fp32 sums of a few hundred
    terms in another order, through two layers: far below 2^-12 of the logits' size."""
    from linear_lm import LinearLM, decode
    torch.manual_seed(0)
    model = LinearLM(300, 128, 2, 1, 2, 64).to(dev)
    ids = torch.randint(0, 300, (2, 90), device=dev)
    out = list(decode(model, ids, 6))
    tokens = torch.stack([t for t, _ in out], 1)
    with torch.no_grad():
        logits, _ = model(torch.cat([ids, tokens[:, :-1]], 1))
    want = torch.log_softmax(logits[:, -6:].double(), -1)
    got = torch.stack([r.logp for _, r in out], 1).double()
    assert torch.equal(torch.stack([r.top_ids[:, 0] for _, r in out], 1), tokens)
    assert float((got - want.gather(-1, tokens[..., None])[..., 0]).abs().max()) < 2 ** -12 * float(logits.abs().max())
    ent = -(want.exp() * want).sum(-1)
    assert float((torch.stack([r.entropy for _, r in out], 1) - ent).abs().max()) < 2 ** -12 * float(logits.abs().max())


@pytest.mark.parametrize("bf16", [False, True])
def test_training_steps(dev, bf16, capsys):
    """The command runs, and repeated steps on one sequence lower its loss."""
    import linear_lm
    assert linear_lm.main(["--steps", "6", "--tokens", "200", "--decode", "3"] + (["--bf16"] if bf16 else [])) == 0
    lines = capsys.readouterr().out.splitlines()
    losses = [float(l.split()[3]) for l in lines if l.startswith("step")]
    assert len(losses) == 6 and losses[-1] < losses[0] - 0.1
    assert sum(l.startswith("token") for l in lines) == 3


def test_gradients_equal_those_of_plain_operators(dev):
    """One step's gradients against the same model with the operators in plain fp64 form.  The model's own products are fp32
    here (2^-24 each, sums of a thousand terms): 2^-12 of a whole gradient's norm is far above both sides' rounding."""
    import linear_lm
    torch.manual_seed(1)
    model = linear_lm.LinearLM(200, 64, 2, 1, 2, 32).to(dev)
    ids = torch.randint(0, 200, (2, 71), device=dev)
    logits, _ = model(ids[:, :-1])
    loss = -linear_lm.token_logprobs(logits, ids[:, 1:]).logp.mean()
    grads = torch.autograd.grad(loss, list(model.parameters()))

    def plain_attention(q, k, v, g, state=None):
        r = v.shape[2] // q.shape[2]
        q, k = q.repeat_interleave(r, 2), k.repeat_interleave(r, 2)
        S, ys = torch.zeros(*v.shape[:1], *v.shape[2:], q.shape[-1], dtype=v.dtype, device=dev), []
        for t in range(q.shape[1]):
            S = S * g[:, t].exp()[..., None, None] + v[:, t, :, :, None] * k[:, t, :, None, :]
            ys.append((S * q[:, t, :, None, :]).sum(-1) * q.shape[-1] ** -0.5)
        return torch.stack(ys, 1), S

    def plain_rotary(q, k, pos, inv):
        ang = pos.double()[:, None] * inv
        c, s = ang.cos()[:, None], ang.sin()[:, None]
        n = inv.numel()
        turn = lambda x: torch.cat([x[..., :n] * c - x[..., n:2 * n] * s, x[..., n:2 * n] * c + x[..., :n] * s,  # noqa: E731
                                    x[..., 2 * n:]], -1)
        return turn(q), turn(k)

    saved = linear_lm.linear_attention, linear_lm.rotary
    try:
        linear_lm.linear_attention, linear_lm.rotary = plain_attention, plain_rotary
        m64 = linear_lm.LinearLM(200, 64, 2, 1, 2, 32).to(dev).double()
        m64.load_state_dict({k: v.double() for k, v in model.state_dict().items()})
        lp = torch.log_softmax(m64(ids[:, :-1])[0], -1).gather(-1, ids[:, 1:, None])
        want = torch.autograd.grad(-lp.mean(), list(m64.parameters()))
    finally:
        linear_lm.linear_attention, linear_lm.rotary = saved
    for (name, _), a, b in zip(model.named_parameters(), grads, want):
        assert float((a.double() - b).norm()) <= 2 ** -12 * float(b.norm()) + 1e-12, name
