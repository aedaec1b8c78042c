"""Operators of a linear-attention language model: the calls that a training step and a decode loop make of them, in
plain form (elementary torch operations in 32 bits, 64 where sums are long or angles large) and as the framework's own
calls.

A case's ``kind`` names the operator:

  attend     linear attention with a decay for each head over whole sequences: forward only (a prompt), or forward and
             backward with every gradient (``train``).  ``decay`` is "token" (a log decay per token and head) or "head"
             (one per head); ``fused``: q, k and v are views of one projection's output.
  step       one token of B sequences, the states updated in place.
  rotary     rotary positions on q and k: forward, or forward and backward (``train``).
  logprobs   log probabilities of given tokens, with entropy and the top alternatives, and with ``train`` the gradient
             of the logits.
  clip       the norm over all gradients of a model, and the gradients scaled by it.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_PKG = str(Path(__file__).resolve().parent.parent / "moe-stream-mac_amd")
DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def _attend(name, **kw):
    c = dict(name=name, kind="attend", B=1, T=64, Hk=16, Hv=32, Dk=128, Dv=128, dtype="bf16", decay="token",
             state=False, train=True, fused=False)
    c.update(kw)
    return c


def listed():
    return [
        # the benchmark's batch and heads, a learned decay per token: one layer of a training step
        _attend("attend_train_bf16_b4_t4096", B=4, T=4096),
        # fp32 training from a carried state (its gradient too), a learned decay per head, an odd length
        _attend("attend_train_fp32_b1_t2047", T=2047, dtype="fp32", decay="head", state=True),
        # two long prompts: forward only, fixed decays, q, k and v views of the projection
        _attend("attend_prompt_bf16_b2_t8100", B=2, T=8100, decay="head", train=False, fused=True),
        # one token of a serving batch, states updated in place
        dict(name="step_bf16_b64", kind="step", B=64, Hk=16, Hv=32, Dk=128, Dv=128, dtype="bf16", decay="token"),
        # the loss of a training step: every token's log probability and the logits' gradient, padding ignored
        dict(name="logprobs_train_bf16_8192x32000", kind="logprobs", N=8192, V=32000, dtype="bf16", train=True,
             entropy=False, top=0, ignored=True, masked=False),
        # a policy's loss with an entropy term: few rows, odd sizes, fp32 logits
        dict(name="logprobs_train_fp32_513x50001", kind="logprobs", N=513, V=50001, dtype="fp32", train=True,
             entropy=True, top=0, ignored=True, masked=True),
        # scoring a batch of sampled tokens: entropy and twenty alternatives of each
        dict(name="logprobs_score_bf16_64x131072", kind="logprobs", N=64, V=131072, dtype="bf16", train=False,
             entropy=True, top=20, ignored=False, masked=True),
        # one sampled token of one sequence: what an interactive user waits for
        dict(name="logprobs_score_bf16_1x131072", kind="logprobs", N=1, V=131072, dtype="bf16", train=False,
             entropy=True, top=5, ignored=False, masked=False),
        # positions of a training step: half layout, part of each head, views of the projection
        dict(name="rotary_train_bf16_b2_t8192", kind="rotary", B=2, T=8192, Hq=32, Hk=16, D=128, R=64, dtype="bf16",
             interleaved=False, train=True, fused=True, start=0, scaled=False),
        # one token of a serving batch far into its sequences: interleaved, frequencies scaled for a long context
        dict(name="rotary_step_bf16_b64", kind="rotary", B=64, T=1, Hq=32, Hk=16, D=128, R=128, dtype="bf16",
             interleaved=True, train=False, fused=False, start=1000000, scaled=True),
        # the gradients of LoRA adapters: many small tensors
        dict(name="clip_fp32_lora", kind="clip", layers=32, hidden=2048, inter=8192, rank=16, dtype="fp32", norm="2"),
        # the gradients of a whole small model: few large tensors
        dict(name="clip_bf16_model", kind="clip", layers=12, hidden=2048, inter=8192, rank=0, dtype="bf16", norm="2"),
    ]


def _logint(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["attend"] * 4 + ["step"] + ["logprobs"] * 3 + ["rotary"] * 2 + ["clip"] * 2)
    Hk, Hv = rng.choice([(16, 32), (16, 32), (16, 16), (8, 16), (4, 16), (3, 6), (1, 5)])
    Dk, Dv = rng.choice([(128, 128)] * 3 + [(64, 64), (64, 128), (128, 64), (96, 96), (32, 48), (256, 256), (80, 33)])
    if kind == "attend":
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp32", "fp16"])
        cap = min(16384, 16384 * 32 * 128 * 128 // (Hv * Dk * Dv * (1 if dtype == "bf16" else 2)))
        B = rng.choice([1, 1, 2, 3, 4, 8])
        T = _logint(rng, 1, max(1, cap // B))
        train = rng.random() < 0.7
        decay = rng.choice(["token", "head"]) if dtype == "fp32" or not train else "token"
        return dict(kind=kind, B=B, T=T, Hk=Hk, Hv=Hv, Dk=Dk, Dv=Dv, dtype=dtype, decay=decay,
                    state=rng.random() < 0.4, train=train, fused=rng.random() < 0.4)
    if kind == "step":
        B = _logint(rng, 1, max(1, 64 * 32 * 128 * 128 // (Hv * Dk * Dv)))
        return dict(kind=kind, B=min(B, 256), Hk=Hk, Hv=Hv, Dk=Dk, Dv=Dv, dtype=rng.choice(["bf16", "fp32", "fp16"]),
                    decay=rng.choice(["token", "head"]))
    if kind == "logprobs":
        train = rng.random() < 0.5
        V = _logint(rng, 1000, 131072)
        most = min(8192, (8192 * 32000 if train else 64 * 131072) // V)
        return dict(kind=kind, N=_logint(rng, 1, max(1, most)), V=V,
                    dtype=rng.choice(["bf16", "bf16", "fp32", "fp16"] if not train else ["bf16", "bf16", "fp32"]),
                    train=train, entropy=rng.random() < 0.5, top=0 if train else rng.choice([0, 1, 5, 20, 32]),
                    ignored=rng.random() < 0.5, masked=rng.random() < 0.4)
    if kind == "rotary":
        B = rng.choice([1, 2, 4, 64])
        D = rng.choice([128, 128, 64, 96, 256])
        Hq = rng.choice([32, 16, 8, 5])
        T = 1 if B == 64 else _logint(rng, 1, 8192 * 128 // (B * D))
        return dict(kind=kind, B=B, T=T, Hq=Hq, Hk=rng.choice([Hq, max(1, Hq // 2), 1]), D=D,
                    R=rng.choice([D, D // 2, D // 4]), dtype=rng.choice(["bf16", "bf16", "fp32", "fp16"]),
                    interleaved=rng.random() < 0.5, train=rng.random() < 0.5, fused=rng.random() < 0.5,
                    start=rng.choice([0, 0, 4096, 1000000]), scaled=rng.random() < 0.5)
    rank = rng.choice([0, 8, 16, 64])
    return dict(kind=kind, layers=_logint(rng, 1, 8 if rank == 0 else 48), hidden=rng.choice([512, 1001, 2048]),
                inter=rng.choice([1024, 4099, 8192]), rank=rank, dtype=rng.choice(["bf16", "fp32", "fp16"]),
                norm=rng.choice(["2", "2", "inf"]))


# ------------------------------------------------------------------------------------------------ inputs


def _clip_shapes(c):
    h, i, r = c["hidden"], c["inter"], c["rank"]
    mats = [(i, h), (i, h), (h, i), (h, h), (h, h)]
    one = [s for m in mats for s in (((r, m[1]), (m[0], r)) if r else (m,))]
    return (one + ([] if r else [(h,), (h,)])) * c["layers"]


def _frequencies(c):
    """Inverse frequencies (64 bits) and the factor on the rotated values; ``scaled``: fast turns kept, slow ones slowed
    eightfold, blended between (positions beyond the trained length)."""
    inv = 10000.0 ** (-torch.arange(0, c["R"], 2, device=DEV, dtype=torch.float64) / c["R"])
    if not c["scaled"]:
        return inv, 1.0
    turns = 4096 * inv / (2 * math.pi)
    keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
    return inv / 8.0 * (1 - keep) + inv * keep, 0.1 * math.log(8.0) + 1.0


def _views(gen, B, T, heads, dtype, fused):
    """N(0, 1) tensors [B, T, H, D], as views of one buffer when fused."""
    if fused:
        x = torch.randn(B, T, sum(h * d for h, d in heads), device=DEV, generator=gen).to(dtype)
        return [p.unflatten(-1, hd) for p, hd in zip(x.split([h * d for h, d in heads], -1), heads)]
    return [torch.randn(B, T, h, d, device=DEV, generator=gen).to(dtype) for h, d in heads]


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))
    rand = lambda *s: torch.randn(*s, device=DEV, generator=gen)  # noqa: E731
    s = {"case": c}
    if c["kind"] in ("attend", "step"):
        B, Hk, Hv, Dk, Dv, dtype = c["B"], c["Hk"], c["Hv"], c["Dk"], c["Dv"], DT[c["dtype"]]
        T = c.get("T", 1)
        q, k, v = _views(gen, B, T, [(Hk, Dk), (Hk, Dk), (Hv, Dv)], dtype, c.get("fused", False))
        rates = torch.exp2(-torch.linspace(1.0, 8.0, Hv, device=DEV))  # memories of a few tokens to hundreds
        if c["decay"] == "head":
            g = -rates * (1 + 0.1 * rand(Hv).abs())
        else:
            g = (-rates * torch.nn.functional.softplus(rand(B, T, Hv))).to(dtype)
        if c["kind"] == "step":
            s.update(q=q[:, 0].contiguous(), k=k[:, 0].contiguous(), v=v[:, 0].contiguous(),
                     g=g if c["decay"] == "head" else g[:, 0].contiguous(), state=rand(B, Hv, Dv, Dk))
            return s
        s.update(q=q, k=k, v=v, g=g, state=0.3 * rand(B, Hv, Dv, Dk) if c["state"] else None)
        if c["train"]:
            s.update(dy=rand(B, T, Hv, Dv).to(dtype), dstate=0.3 * rand(B, Hv, Dv, Dk))
            for n in ("q", "k", "v", "g", "state"):
                if s[n] is not None:
                    s[n] = s[n].detach().requires_grad_(True)
    elif c["kind"] == "rotary":
        B, T, dtype = c["B"], c["T"], DT[c["dtype"]]
        heads = [(c["Hq"], c["D"]), (c["Hk"], c["D"])]
        q, k = _views(gen, B, T, heads, dtype, c["fused"])
        off = torch.randint(0, 4096, (B, 1), device=DEV, generator=gen) if T == 1 else 0
        inv, factor = _frequencies(c)
        s.update(q=q, k=k, positions=c["start"] + off + torch.arange(T, device=DEV).expand(B, T), inv=inv, factor=factor)
        if c["train"]:
            dq, dk = _views(gen, B, T, heads, dtype, False)
            s.update(q=q.detach().requires_grad_(True), k=k.detach().requires_grad_(True), dq=dq, dk=dk)
    elif c["kind"] == "logprobs":
        N, V = c["N"], c["V"]
        z = 3.0 * rand(N, V)
        target = torch.randint(0, V, (N,), device=DEV, generator=gen)
        if c["masked"]:  # tokens that the sampler's grammar bans
            ban = torch.rand(N, V, device=DEV, generator=gen) < 0.3
            ban[torch.arange(N, device=DEV), target] = False
            z = z.masked_fill(ban, float("-inf"))
        if c["ignored"]:
            target = target.masked_fill(torch.rand(N, device=DEV, generator=gen) < 0.2, -100)
        s.update(logits=z.to(DT[c["dtype"]]), target=target)
        if c["train"]:
            s.update(logits=s["logits"].requires_grad_(True), dlogp=rand(N) / N, dent=rand(N) / N)
    else:
        shapes = _clip_shapes(c)
        sizes = [math.prod(x) for x in shapes]
        flat = torch.empty(sum(sizes), device=DEV, dtype=DT[c["dtype"]])
        for part, size in zip(flat.split(1 << 26), range(0, flat.numel(), 1 << 26)):
            part.copy_(0.02 * rand(part.numel()))
        out = torch.empty_like(flat)
        cut = lambda x: [p.view(sh) for p, sh in zip(x.split(sizes), shapes)]  # noqa: E731
        s.update(flat=out, grads=cut(flat), out=cut(out), max_norm=1.0 if c["norm"] == "2" else 0.01)
    return s


# ------------------------------------------------------------------------------------------------ plain forms


def _plain_attend(q, k, v, g, state, scale):
    """Chunks of 64 tokens: products inside each, their states joined by one product with the decays between chunks."""
    B, T, Hk, Dk = q.shape
    Hv, Dv = v.shape[2], v.shape[3]
    N = max(1, -(-T // 64))

    def lay(x):  # [B, T, H, D] -> [B, Hv, N, 64, D], zeros after the end
        x = x.float().repeat_interleave(Hv // x.shape[2], dim=2)
        return torch.nn.functional.pad(x, (0, 0, 0, 0, 0, N * 64 - T)).unflatten(1, (N, 64)).permute(0, 3, 1, 2, 4)

    q, k, v = lay(q) * scale, lay(k), lay(v)
    g = torch.nn.functional.pad(g.double().expand(B, T, Hv), (0, 0, 0, N * 64 - T))
    G = g.unflatten(1, (N, 64)).permute(0, 3, 1, 2).cumsum(-1)  # decays add up in 64 bits
    end = G[..., -1].cumsum(-1)
    start = torch.cat([end - G[..., -1], end[..., -1:]], -1)
    low = torch.ones(64, 64, dtype=torch.bool, device=q.device).tril()
    inside = (G[..., :, None] - G[..., None, :]).masked_fill(~low, float("-inf")).exp().float()
    before = torch.ones(N + 1, N, dtype=torch.bool, device=q.device).tril(-1)
    across = (start[..., :, None] - end[..., None, :]).masked_fill(~before, float("-inf")).exp().float()
    add = (k * (G[..., -1:] - G).exp().float()[..., None]).transpose(-1, -2) @ v
    S = (across @ add.flatten(-2)).unflatten(-1, (Dk, Dv))
    if state is not None:
        S = S + start.exp().float()[..., None, None] * state.transpose(-1, -2)[:, :, None]
    y = ((q @ k.transpose(-1, -2)) * inside) @ v + G.exp().float()[..., None] * (q @ S[:, :, :N])
    y = y.permute(0, 2, 3, 1, 4).flatten(1, 2)[:, :T]
    return y, S[:, :, N].transpose(-1, -2).contiguous()


def _rotate(x, cos, sin, R, interleaved):
    x32 = x.float()
    a, b = (x32[..., 0:R:2], x32[..., 1:R:2]) if interleaved else (x32[..., :R // 2], x32[..., R // 2:R])
    ra, rb = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([ra, rb], -1).flatten(-2) if interleaved else torch.cat([ra, rb], -1)
    return torch.cat([turned, x32[..., R:]], -1).to(x.dtype)


def run(state):
    s, c = state, state["case"]
    if own:
        return _run_own(s, c)
    kind = c["kind"]
    if kind == "attend":
        names = [n for n in ("q", "k", "v", "g", "state") if s[n] is not None]
        y, last = _plain_attend(s["q"], s["k"], s["v"], s["g"], s["state"], c["Dk"] ** -0.5)
        y = y.to(s["q"].dtype)
        out = {"y": y, "last": last}
        if c["train"]:
            out["grads"] = dict(zip(names, torch.autograd.grad([y, last], [s[n] for n in names], [s["dy"], s["dstate"]])))
        return out
    if kind == "step":
        r = c["Hv"] // c["Hk"]
        q, k, v = s["q"].float().repeat_interleave(r, 1), s["k"].float().repeat_interleave(r, 1), s["v"].float()
        S = s["state"] * s["g"].float().exp().expand(c["B"], -1)[..., None, None] + v[..., None] * k[..., None, :]
        s["state"].copy_(S)
        return {"y": ((S * q[..., None, :]).sum(-1) * c["Dk"] ** -0.5).to(s["v"].dtype), "state": s["state"]}
    if kind == "rotary":
        angle = (s["positions"].double()[..., None] * s["inv"])[:, :, None]
        cos, sin = (angle.cos() * s["factor"]).float(), (angle.sin() * s["factor"]).float()
        out = {n: _rotate(s[n].detach(), cos, sin, c["R"], c["interleaved"]) for n in ("q", "k")}
        if c["train"]:  # the rotation back; the rest of a head passes through
            out.update({n: _rotate(s[n], cos, -sin, c["R"], c["interleaved"]) for n in ("dq", "dk")})
        return out
    if kind == "logprobs":
        z = s["logits"].detach().float()
        gone = z == float("-inf")
        top = z.max(-1, keepdim=True).values
        e = (z - top).exp()
        total = e.sum(-1, keepdim=True)
        logp = z - top - total.log()
        p = e / total
        ent = -(p * logp.masked_fill(gone, 0.0)).sum(-1)
        live = s["target"] != -100
        at = s["target"].clamp_min(0)[:, None]
        out = {"logp": logp.gather(-1, at)[:, 0].masked_fill(~live, 0.0)}
        if c["entropy"]:
            out["entropy"] = ent
        if c["top"]:  # equal values in the order of their indices
            ids = torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :c["top"]]
            out["ids"], out["top"] = ids, logp.gather(-1, ids)
        if c["train"]:
            d = (s["dlogp"] * live)[:, None]
            dz = -d * p
            dz.scatter_add_(-1, at, d)
            if c["entropy"]:
                dz = dz - s["dent"][:, None] * p * (logp.masked_fill(gone, 0.0) + ent[:, None])
            out["dlogits"] = dz.to(s["logits"].dtype)
        return out
    if c["norm"] == "2":
        norm = torch.stack([x.float().square().sum(dtype=torch.float64) for x in s["grads"]]).sum().sqrt().float()
    else:
        norm = torch.stack([x.float().abs().max() for x in s["grads"]]).max()
    factor = (s["max_norm"] / (norm + 1e-6)).clamp_max(1.0)
    torch.cat([(x.float() * factor).to(x.dtype).flatten() for x in s["grads"]], out=s["flat"])
    return {"norm": norm, "grads": s["flat"]}


# ------------------------------------------------------------------------------------------------ the framework's calls


def _run_own(s, c):
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    kind = c["kind"]
    if kind == "attend":
        from linear_attention import linear_attention
        names = [n for n in ("q", "k", "v", "g", "state") if s[n] is not None]
        y, last = linear_attention(s["q"], s["k"], s["v"], s["g"], s["state"])
        out = {"y": y, "last": last}
        if c["train"]:
            out["grads"] = dict(zip(names, torch.autograd.grad([y, last], [s[n] for n in names], [s["dy"], s["dstate"]])))
        return out
    if kind == "step":
        from linear_attention import linear_attention_step
        y = linear_attention_step(s["q"], s["k"], s["v"], s["g"], s["state"])
        return {"y": y, "state": s["state"]}
    if kind == "rotary":
        from rotary import rotary
        q, k = rotary(s["q"], s["k"], s["positions"], s["inv"], interleaved=c["interleaved"], factor=s["factor"])
        out = {"q": q, "k": k}
        if c["train"]:
            out["dq"], out["dk"] = torch.autograd.grad([q, k], [s["q"], s["k"]], [s["dq"], s["dk"]])
        return out
    if kind == "logprobs":
        from token_logprobs import token_logprobs
        r = token_logprobs(s["logits"], s["target"], entropy=c["entropy"], top=c["top"])
        out = {"logp": r.logp}
        if c["entropy"]:
            out["entropy"] = r.entropy
        if c["top"]:
            out["ids"], out["top"] = r.top_ids, r.top_logp
        if c["train"]:
            heads = [(r.logp, s["dlogp"])] + ([(r.entropy, s["dent"])] if c["entropy"] else [])
            out["dlogits"] = torch.autograd.grad([h for h, _ in heads], [s["logits"]], [d for _, d in heads])[0]
        return out
    from grad_clip import clip_grad_norm
    norm = clip_grad_norm(s["grads"], s["max_norm"], 2.0 if c["norm"] == "2" else math.inf, out=s["out"])
    return {"norm": norm, "grads": s["flat"]}


# ------------------------------------------------------------------------------------------------ work


def work(case):
    c = case
    e = SIZE[c["dtype"]]
    if c["kind"] in ("attend", "step"):
        B, T, Hk, Hv, Dk, Dv = c["B"], c.get("T", 1), c["Hk"], c["Hv"], c["Dk"], c["Dv"]
        qk, vo, st = B * T * Hk * Dk * e, B * T * Hv * Dv * e, B * Hv * Dk * Dv * 4
        g = Hv * 4 if c["decay"] == "head" else B * T * Hv * e
        flops = 4 * B * T * Hv * Dk * Dv
        if c["kind"] == "step":
            return {"bytes": 2 * qk + 2 * vo + g + 2 * st, "flops": flops}
        fwd = 2 * qk + 2 * vo + g + st * (2 if c["state"] else 1)
        if not c["train"]:
            return {"bytes": fwd, "flops": flops}
        return {"bytes": fwd + vo + st + 2 * qk + vo + g + (st if c["state"] else 0), "flops": 3 * flops}
    if c["kind"] == "rotary":
        x = c["B"] * c["T"] * (c["Hq"] + c["Hk"]) * c["D"] * e
        n = 2 if c["train"] else 1
        return {"bytes": n * 2 * x + c["B"] * c["T"] * 8, "flops": n * 3 * x / e}
    if c["kind"] == "logprobs":
        x, out = c["N"] * c["V"] * e, c["N"] * (4 + 4 + 8 + 12 * c["top"])
        n = c["N"] * c["V"] * (5 + (5 if c["train"] else 0))
        return {"bytes": x * (2 if c["train"] else 1) + out, "flops": n}
    n = sum(math.prod(x) for x in _clip_shapes(c))
    return {"bytes": 2 * n * e, "flops": 3 * n}


# ------------------------------------------------------------------------------------------------ 64 bits


def _exact_attend(s, c):
    """The recurrence token by token: the forward with dq, then the reverse with dk, dv and dg."""
    B, T, Hv, r = c["B"], c["T"], c["Hv"], c["Hv"] // c["Hk"]
    d = lambda n: s[n].detach().double()  # noqa: E731
    q = d("q").repeat_interleave(r, 2).transpose(0, 1).contiguous() * c["Dk"] ** -0.5
    k = d("k").repeat_interleave(r, 2).transpose(0, 1).contiguous()
    v = d("v").transpose(0, 1).contiguous()
    g = d("g").expand(B, T, Hv).transpose(0, 1).contiguous()
    a = g.exp()[..., None, None]
    S = d("state") if s["state"] is not None else torch.zeros(B, Hv, c["Dv"], c["Dk"], device=DEV, dtype=torch.float64)
    y, dq = torch.empty_like(v), torch.empty_like(q)
    dy = d("dy").transpose(0, 1).contiguous() if c["train"] else None
    for t in range(T):
        S = a[t] * S + v[t][..., None] * k[t][..., None, :]
        y[t] = (S * q[t][..., None, :]).sum(-1)
        if c["train"]:
            dq[t] = (S * dy[t][..., None]).sum(-2)
    out = {"y": y.transpose(0, 1), "last": S}
    if not c["train"]:
        return out
    dS, dk, dv = d("dstate").clone(), torch.empty_like(k), torch.empty_like(v)
    tail = (dS * S).sum((-1, -2))
    for t in range(T - 1, -1, -1):
        dS = dS + dy[t][..., None] * q[t][..., None, :]
        dk[t] = (dS * v[t][..., None]).sum(-2)
        dv[t] = (dS * k[t][..., None, :]).sum(-1)
        dS = a[t] * dS
    per = (q * dq).sum(-1) - (k * dk).sum(-1)  # the gradient of the summed log decays
    dg = per.flip(0).cumsum(0).flip(0) + tail
    fold = lambda x: x.transpose(0, 1).unflatten(2, (c["Hk"], r)).sum(3)  # noqa: E731
    out["grads"] = {"q": fold(dq) * c["Dk"] ** -0.5, "k": fold(dk), "v": dv.transpose(0, 1),
                    "g": dg.sum((0, 1)) if c["decay"] == "head" else dg.transpose(0, 1)}
    if s["state"] is not None:
        out["grads"]["state"] = dS
    return out


def exact(case, seed):
    c, s = case, prepare(case, seed)
    kind = c["kind"]
    if kind == "attend":
        return _exact_attend(s, c)
    if kind == "step":
        r = c["Hv"] // c["Hk"]
        q, k = (s[n].double().repeat_interleave(r, 1) for n in ("q", "k"))
        S = torch.einsum("bhv,bhk->bhvk", s["v"].double(), k)
        S += s["state"].double() * torch.exp(s["g"].double()).expand(c["B"], -1)[:, :, None, None]
        return {"y": (S @ q[..., None])[..., 0] / math.sqrt(c["Dk"]), "state": S}
    if kind == "rotary":
        turn = torch.polar(torch.full((), s["factor"], device=DEV, dtype=torch.float64),
                           s["positions"].double()[:, :, None, None] * s["inv"])

        def rot(x, by):
            x, h = x.detach().double(), c["R"] // 2
            part = x[..., :c["R"]]
            pair = part.unflatten(-1, (h, 2)) if c["interleaved"] else part.unflatten(-1, (2, h)).transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * by)
            z = z if c["interleaved"] else z.transpose(-1, -2)
            return torch.cat([z.flatten(-2), x[..., c["R"]:]], -1)

        out = {n: rot(s[n], turn) for n in ("q", "k")}
        if c["train"]:
            out.update({n: rot(s[n], turn.conj()) for n in ("dq", "dk")})
        return out
    if kind == "logprobs":
        z = s["logits"].detach().double()
        logp = z - torch.logsumexp(z, -1, keepdim=True)
        p = logp.exp()
        plogp = torch.where(p > 0, p * logp, torch.zeros_like(p))
        ent = -plogp.sum(-1)
        live = s["target"] >= 0
        rows = torch.arange(c["N"], device=DEV)
        at = torch.where(live, s["target"], torch.zeros_like(s["target"]))
        out = {"logp": torch.where(live, logp[rows, at], torch.zeros_like(ent))}
        if c["entropy"]:
            out["entropy"] = ent
        if c["top"]:
            out["ids"], out["top"] = None, torch.topk(logp, c["top"], -1).values
        if c["train"]:
            d = s["dlogp"].double() * live
            dz = p * -d[:, None]
            dz[rows, at] += d
            if c["entropy"]:
                dz -= s["dent"].double()[:, None] * (plogp + p * ent[:, None])
            out["dlogits"] = dz
        return out
    total = [x.double() for x in s["grads"]]
    if c["norm"] == "2":
        norm = math.sqrt(sum(float((x * x).sum()) for x in total))
    else:
        norm = max(float(x.abs().max()) for x in total)
    by = min(1.0, s["max_norm"] / (norm + 1e-6))
    return {"norm": torch.tensor(norm, dtype=torch.float64), "grads": torch.cat([(x * by).flatten() for x in total])}
