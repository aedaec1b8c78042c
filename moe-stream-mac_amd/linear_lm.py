"""A small language model of linear-attention layers, trained for a few steps and then decoded token by token: the
operators of ``linear_attention``, ``rotary``, ``token_logprobs`` and ``grad_clip`` as one program uses them.

    python moe-stream-mac_amd/linear_lm.py --steps 4 --tokens 512 --decode 16

The model is random-initialised and trained with AdamW on synthetic next-token data.  Prints the loss and the gradients'
norm of every step, then for every decoded token its log probability, the entropy it was drawn from and its best
alternative.
"""

from __future__ import annotations

import argparse
import sys
import time
from typing import Optional

import torch
import torch.nn.functional as F

from grad_clip import clip_grad_norm
from linear_attention import linear_attention, linear_attention_step
from rotary import rotary, rotary_frequencies
from token_logprobs import token_logprobs

Array = torch.Tensor


class Mixer(torch.nn.Module):
    """Linear attention over one projection's q, k, v and log decays (one per token and value head)."""

    def __init__(self, hidden: int, key_heads: int, value_heads: int, head_dim: int):
        super().__init__()
        self.heads = (key_heads, value_heads, head_dim)
        self.sizes = [key_heads * head_dim, key_heads * head_dim, value_heads * head_dim, value_heads]
        self.proj = torch.nn.Linear(hidden, sum(self.sizes), bias=False)
        self.out = torch.nn.Linear(value_heads * head_dim, hidden, bias=False)
        # memories of a few tokens to hundreds
        self.rate = torch.nn.Parameter(-torch.linspace(0.7, 5.5, value_heads))

    def forward(self, x: Array, positions: Array, inv_freq: Array, state: Optional[Array]) -> tuple[Array, Array]:
        Hk, Hv, D = self.heads
        q, k, v, a = self.proj(x).split(self.sizes, -1)
        q, k, v = q.unflatten(-1, (Hk, D)), k.unflatten(-1, (Hk, D)), v.unflatten(-1, (Hv, D))
        q, k = rotary(F.normalize(q, dim=-1) * D ** 0.5, F.normalize(k, dim=-1), positions, inv_freq)
        g = -self.rate.exp() * F.softplus(a)
        if x.shape[1] == 1 and state is not None and not torch.is_grad_enabled():  # one token: the state in place
            y = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], state)[:, None]
        else:
            y, state = linear_attention(q, k, v, g, state)
        return self.out(y.flatten(-2)), state


class LinearLM(torch.nn.Module):
    def __init__(self, vocab: int, hidden: int, layers: int, key_heads: int, value_heads: int, head_dim: int):
        super().__init__()
        self.embed = torch.nn.Embedding(vocab, hidden)
        self.norms = torch.nn.ModuleList(torch.nn.LayerNorm(hidden) for _ in range(2 * layers + 1))
        self.mixers = torch.nn.ModuleList(Mixer(hidden, key_heads, value_heads, head_dim) for _ in range(layers))
        self.mlps = torch.nn.ModuleList(
            torch.nn.Sequential(torch.nn.Linear(hidden, 4 * hidden), torch.nn.GELU(), torch.nn.Linear(4 * hidden, hidden))
            for _ in range(layers))
        self.head = torch.nn.Linear(hidden, vocab, bias=False)
        self.register_buffer("inv_freq", rotary_frequencies(head_dim // 2)[0], persistent=False)

    def _apply(self, fn, *args, **kw):
        """Moves and casts of the whole model: the frequencies go along and keep their 64 bits."""
        inv = self.inv_freq
        super()._apply(fn, *args, **kw)
        self.inv_freq = inv.to(self.inv_freq.device)
        return self

    def forward(self, ids: Array, start: int = 0, states: Optional[list] = None) -> tuple[Array, list]:
        """(logits [B, T, vocab], the layers' states after the last token) of ids [B, T] at positions start on."""
        positions = torch.arange(start, start + ids.shape[1], device=ids.device)
        x, out = self.embed(ids), []
        for i, (mixer, mlp) in enumerate(zip(self.mixers, self.mlps)):
            y, state = mixer(self.norms[2 * i](x), positions, self.inv_freq, None if states is None else states[i])
            out.append(state)
            x = x + y
            x = x + mlp(self.norms[2 * i + 1](x))
        return self.head(self.norms[-1](x)), out


def train_step(model: LinearLM, opt, ids: Array, max_norm: float) -> tuple[Array, Array]:
    """(loss, the gradients' norm before clipping) of one step on ids [B, T + 1]."""
    logits, _ = model(ids[:, :-1])
    loss = -token_logprobs(logits, ids[:, 1:]).logp.mean()
    opt.zero_grad(set_to_none=True)
    loss.backward()
    norm = clip_grad_norm([p.grad for p in model.parameters() if p.grad is not None], max_norm)
    opt.step()
    return loss.detach(), norm


@torch.no_grad()
def decode(model: LinearLM, prompt: Array, tokens: int):
    """Greedy tokens after prompt [B, T], one at a time: yields (ids [B], their TokenLogprobs with two alternatives)."""
    logits, states = model(prompt)
    for i in range(tokens):
        last = logits[:, -1]
        ids = last.argmax(-1)
        yield ids, token_logprobs(last, ids, entropy=True, top=2)
        if i + 1 < tokens:
            logits, states = model(ids[:, None], prompt.shape[1] + i, states)


def main(argv: list[str] | None = None) -> int:
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--steps", type=int, default=4)
    p.add_argument("--batch", type=int, default=1)
    p.add_argument("--tokens", type=int, default=512)
    p.add_argument("--decode", type=int, default=8)
    p.add_argument("--hidden", type=int, default=256)
    p.add_argument("--layers", type=int, default=2)
    p.add_argument("--key-heads", type=int, default=2)
    p.add_argument("--value-heads", type=int, default=4)
    p.add_argument("--head-dim", type=int, default=64)
    p.add_argument("--vocab", type=int, default=1000)
    p.add_argument("--lr", type=float, default=1e-3)
    p.add_argument("--max-norm", type=float, default=1.0)
    p.add_argument("--bf16", action="store_true")
    p.add_argument("--seed", type=int, default=0)
    args = p.parse_args(argv)
    if args.steps < 0 or args.tokens < 1 or args.decode < 0:
        p.error("steps and decode must not be negative, tokens at least 1")
    if not torch.cuda.is_available():
        print("linear_lm needs a ROCm GPU", file=sys.stderr)
        return 1
    dev = torch.device("cuda:0")
    torch.manual_seed(args.seed)
    model = LinearLM(args.vocab, args.hidden, args.layers, args.key_heads, args.value_heads, args.head_dim)
    model = model.to(device=dev, dtype=torch.bfloat16 if args.bf16 else torch.float32)
    opt = torch.optim.AdamW(model.parameters(), lr=args.lr)
    ids = torch.randint(0, args.vocab, (args.batch, args.tokens + 1), device=dev)
    torch.cuda.synchronize(dev)
    started = time.perf_counter()
    for step in range(args.steps):
        loss, norm = train_step(model, opt, ids, args.max_norm)
        print(f"step {step + 1}: loss {loss.item():.4f} gradient norm {norm.item():.4f}", flush=True)
    torch.cuda.synchronize(dev)
    if args.steps:
        print(f"s_per_step={(time.perf_counter() - started) / args.steps:.4f}")
    for i, (tok, r) in enumerate(decode(model, ids[:, :-1], args.decode)):
        print(f"token {i + 1}: id {tok[0].item()} log probability {r.logp[0].item():.4f} entropy {r.entropy[0].item():.4f} "
              f"next best {r.top_ids[0, 1].item()} ({r.top_logp[0, 1].item():.4f})", flush=True)
    return 0


if __name__ == "__main__":
    sys.exit(main())
