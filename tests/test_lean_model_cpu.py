"""What the loss without logits, the sorted embedding and 4-bit layers do to a model that is not plain: kept or refused, never
dropped (no kernel launches)."""

import pytest
import torch
import torch.nn as nn

import mxfp4
import qwen3_5 as Q
from embedding import Embedding


def model():
    torch.manual_seed(0)
    return Q.Model(Q.ModelArgs(hidden_size=32, intermediate_size=64, num_hidden_layers=2, num_attention_heads=2, vocab_size=50,
                               linear_num_key_heads=1, linear_num_value_heads=2, linear_key_head_dim=64,
                               linear_value_head_dim=64, full_attention_interval=2))


def biased(m):
    m.lm_head = nn.Linear(32, 50)


def adapted(m):
    m.lm_head = Q.LoRALinear(m.lm_head, 2, 2.0)


def hooked(m):
    m.lm_head.register_forward_hook(lambda mod, args, out: 2 * out)


def normed(m):
    m.lm_head = nn.utils.parametrizations.weight_norm(m.lm_head)


@pytest.mark.parametrize("change", [biased, adapted, hooked, normed])
def test_loss_takes_plain_heads_only(change):
    """Adapters, a bias, hooks and parametrisations of the head have a part in the logits, which the loss would leave out."""
    m = model()
    change(m)
    ids = torch.zeros(1, 4, dtype=torch.int64)
    with pytest.raises(ValueError, match="bias-free Linear head"):
        m.loss(ids, ids)


def test_sorted_embedding_drops_nothing():
    for kw in (dict(max_norm=1.0), dict(sparse=True), dict(scale_grad_by_freq=True)):
        m = model()
        m.model.embed_tokens = nn.Embedding(50, 32, **kw)
        with pytest.raises(ValueError, match="not supported"):
            Q.sorted_embedding(m)
    m = model()
    m.model.embed_tokens.register_forward_hook(lambda mod, args, out: 2 * out)
    with pytest.raises(ValueError, match="hooks"):
        Q.sorted_embedding(m)
    m = model()
    m.model.embed_tokens = scaled = Embedding(50, 32, scale=3.0)
    Q.sorted_embedding(m)
    assert m.model.embed_tokens is scaled
    m = model()
    old = m.model.embed_tokens = nn.Embedding(50, 32, padding_idx=-1)
    Q.sorted_embedding(m)
    new = m.model.embed_tokens
    assert type(new) is Embedding and new.weight is old.weight and new.padding_idx == 49


def test_four_bits_keep_hooked_layers(monkeypatch):
    q = mxfp4.Weight(torch.zeros(1, 16, dtype=torch.uint8), torch.zeros(1, 1, dtype=torch.uint8), 32)
    monkeypatch.setattr(mxfp4, "quantize", lambda w: q)
    m = model()
    Q.linear_to_lora_layers(m, 1)
    hooked = m.layers[0].gate_up
    hooked.register_forward_hook(lambda mod, args, out: 2 * out)
    count = Q.quantize_frozen(m)
    assert count > 5 and m.layers[0].gate_up is hooked and isinstance(m.layers[0].down, mxfp4.MXFP4Linear)
    assert isinstance(m.layers[1].down.base, mxfp4.MXFP4Linear)
    Q.linear_to_lora_layers(m, 1)  # layers in 4 bits that have their adapters stay
    with pytest.raises(ValueError, match="adapters on first"):
        Q.linear_to_lora_layers(m, 2)


def test_scaled_rows_on_the_cpu_keep_their_bits():
    """The factor meets the rows in 64 bits, as on the GPU."""
    e = Embedding(7, 5, scale=3 ** 0.5, dtype=torch.float64)
    ids = torch.arange(7)
    assert torch.equal(e(ids), e.weight * 3 ** 0.5)
    f = Embedding(7, 5, scale=3 ** 0.5)
    assert torch.equal(f(ids), (f.weight.double() * 3 ** 0.5).float())
