"""GPU checks of the operators of training in little memory as the models use them: the loss without logits, the embedding by
sorted tokens and 4-bit base weights together, against the same models with dense weights and logits.

Both sides are fp32 models of the same formulas: products of a few hundred terms in another order (2^-24 each) through two or
three layers.  2^-12 of a whole gradient's norm is far above both sides' rounding.
"""

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import gdn_lib
    gdn_lib.load()
    return torch.device("cuda:0")


def close(a, b, what):
    assert float((a.double() - b.double()).norm()) <= 2 ** -12 * float(b.double().norm()), what


def test_linear_lm_lean(dev):
    from linear_lm import LinearLM
    torch.manual_seed(0)
    plain = LinearLM(300, 128, 2, 1, 2, 64).to(dev)
    lean = LinearLM(300, 128, 2, 1, 2, 64, lean=True).to(dev)
    lean.load_state_dict(plain.state_dict())
    ids = torch.randint(0, 300, (2, 71), device=dev)
    from linear_lm import linear_cross_entropy
    want = F.cross_entropy(plain(ids[:, :-1])[0].flatten(0, 1), ids[:, 1:].flatten())
    got = linear_cross_entropy(lean.hidden(ids[:, :-1])[0], lean.head.weight, ids[:, 1:])
    close(got, want, "loss")
    names = [n for n, _ in plain.named_parameters()]
    for n, a, b in zip(names, torch.autograd.grad(got, list(lean.parameters())), torch.autograd.grad(want, list(plain.parameters()))):
        close(a, b, n)


def test_tied_weights(dev):
    """One table at both ends: its gradient is the sum of the embedding's and the loss's."""
    from linear_lm import LinearLM, linear_cross_entropy
    torch.manual_seed(1)
    model = LinearLM(200, 64, 1, 1, 2, 32, tied=True).to(dev)
    assert model.head.weight is model.embed.weight and "head.weight" in dict(model.named_parameters(remove_duplicate=False))
    ids = torch.randint(0, 200, (3, 41), device=dev)
    got, = torch.autograd.grad(linear_cross_entropy(model.hidden(ids[:, :-1])[0], model.head.weight, ids[:, 1:]), model.embed.weight)
    scale, model.embed = model.embed.scale, torch.nn.Embedding(200, 64, device=dev)
    model.embed.weight = model.head.weight
    model.embed.register_forward_hook(lambda m, a, y: y * scale)
    want, = torch.autograd.grad(F.cross_entropy(model(ids[:, :-1])[0].flatten(0, 1), ids[:, 1:].flatten()), model.head.weight)
    close(got, want, "tied")


def test_adapters_on_a_4_bit_base(dev):
    """Adapters' gradients over 4-bit layers equal those over dense layers with the same values; ignored targets do not count."""
    import mxfp4
    import qwen3_5 as Q
    torch.manual_seed(2)
    args = Q.ModelArgs(hidden_size=128, intermediate_size=192, num_hidden_layers=3, num_attention_heads=2, vocab_size=300,
                       linear_num_key_heads=1, linear_num_value_heads=2, linear_key_head_dim=64, linear_value_head_dim=64,
                       full_attention_interval=3)
    four = Q.Model(args).to(dev)
    Q.linear_to_lora_layers(four, 2, rank=4)
    four = four.to(dev)
    for n, p in four.named_parameters():
        if "lora_b" in n:
            torch.nn.init.normal_(p, std=0.05)
    import copy
    dense = copy.deepcopy(four)
    for m in dense.modules():
        if type(m) is torch.nn.Linear and m is not dense.lm_head:
            m.weight.data = mxfp4.dequantize(mxfp4.quantize(m.weight), torch.float32)
    Q.sorted_embedding(four)
    linears = sum(type(m) is torch.nn.Linear for layer in four.layers for m in layer.modules())
    assert Q.quantize_frozen(four) == linears and Q.quantize_frozen(four) == 0
    ids = torch.randint(0, 300, (2, 91), device=dev)
    targets = ids[:, 1:].masked_fill(torch.rand(2, 90, device=dev) < 0.3, -100)
    got = four.loss(ids[:, :-1], targets)
    want = F.cross_entropy(dense(ids[:, :-1]).flatten(0, 1), targets.flatten())
    close(got, want, "loss")
    trained = lambda m: [(n, p) for n, p in m.named_parameters() if p.requires_grad]  # noqa: E731
    a, b = trained(four), trained(dense)
    assert [n for n, _ in a] == [n for n, _ in b] and a
    for (n, _), x, y in zip(a, torch.autograd.grad(got, [p for _, p in a]), torch.autograd.grad(want, [p for _, p in b])):
        close(x, y, n)


def test_decoding_on_a_4_bit_base(dev):
    """One token at a time through caches gives the logits of the whole sequence."""
    import qwen3_5 as Q
    torch.manual_seed(3)
    args = Q.ModelArgs(hidden_size=128, intermediate_size=192, num_hidden_layers=2, num_attention_heads=2, vocab_size=100,
                       linear_num_key_heads=1, linear_num_value_heads=2, linear_key_head_dim=64, linear_value_head_dim=64)
    model = Q.Model(args).to(dev).eval()
    Q.freeze(model)
    Q.quantize_frozen(model)
    ids = torch.randint(0, 100, (2, 75), device=dev)
    with torch.no_grad():
        whole = model(ids)
        cache = model.make_cache()
        parts = [model(ids[:, :70], cache=cache)] + [model(ids[:, t:t + 1], cache=cache) for t in range(70, 75)]
    assert float((torch.cat(parts, 1) - whole).abs().max()) < 2 ** -12 * float(whole.abs().max())


@pytest.mark.parametrize("extra", [["--lean"], ["--lean", "--base-bits", "4", "--bf16"], ["--base-bits", "4"]])
def test_lora_step(dev, extra, capsys, monkeypatch):
    import lora_step
    for name in ("GDN_CHECKPOINT", "GDN_VJP", "FROZEN_GDN_KERNEL"):
        monkeypatch.setenv(name, "0")  # installs stay for the process
    assert lora_step.main(["--steps", "2", "--tokens", "100", "--hidden", "128", "--head-dim", "64", *extra]) == 0
    assert sum(l.startswith("step") for l in capsys.readouterr().out.splitlines()) == 2


@pytest.mark.parametrize("extra", [["--lean"], ["--tied", "--bf16"]])
def test_linear_lm_command(dev, extra, capsys):
    import linear_lm
    assert linear_lm.main(["--steps", "2", "--tokens", "100", "--decode", "2", *extra]) == 0
    assert sum(l.startswith("token") for l in capsys.readouterr().out.splitlines()) == 2
