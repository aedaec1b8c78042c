"""Host logic of the example language model (no kernel launches)."""

import torch


def test_frequencies_keep_their_bits():
    """Moved or cast as a whole, the model's rotary frequencies stay float64: rounded to bf16, angles of the thousandth token
    would be off by radians."""
    from linear_lm import LinearLM
    from rotary import rotary_frequencies
    want, _ = rotary_frequencies(16)
    model = LinearLM(10, 16, 1, 1, 2, 32)
    for cast in (model, model.bfloat16(), model.to(dtype=torch.float32), model.half(), model.to("cpu", torch.bfloat16)):
        assert cast.inv_freq.dtype == torch.float64 and torch.equal(cast.inv_freq, want)
    assert model.head.weight.dtype == torch.bfloat16 and "inv_freq" not in model.state_dict()


def test_lean_models_hold_the_same_parameters():
    """A lean model loads a plain one's state; a tied one has a single table at both ends."""
    from linear_lm import LinearLM
    plain, lean = LinearLM(10, 16, 1, 1, 2, 32), LinearLM(10, 16, 1, 1, 2, 32, lean=True)
    lean.load_state_dict(plain.state_dict())
    assert torch.equal(lean.embed(torch.arange(10)), plain.embed.weight)
    tied = LinearLM(10, 16, 1, 1, 2, 32, tied=True)
    assert tied.lean and tied.head.weight is tied.embed.weight and tied.embed.scale == 4.0
    tied = tied.double().float()
    assert tied.head.weight is tied.embed.weight
