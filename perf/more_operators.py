"""Operators of training and decoding in little memory: the loss of a language model whose logits are never kept, the
embedding's gradient by sorted tokens, and frozen weights in microscaled 4-bit floating point; in plain form (elementary
torch operations in 32 bits, 64 where sums are long) and as the framework's own calls.

A case's ``kind`` names the operator:

  loss      cross entropy of the logits x W^T of N tokens over V words.  ``grads``: "" (scores of given tokens), "x" (a
            frozen head, as under LoRA adapters) or "xw".  ``mean``: the mean over the tokens that count, else each
            token's own loss under a weight of its own (``grads``) or as it is.  ``ignored``: a fifth of the tokens do
            not count.
  embed     rows of a table, scaled: forward, or forward and the table's gradient (``train``).  ``padded``: a third of
            the tokens is padding, which has no gradient.
  quantize  a weight in blocks of 32 with a common power of two and 4-bit elements, and the values that these stand for.
  linear    a product with such a weight: forward, or forward and the input's gradient (``train``).
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


def listed():
    return [
        # the loss of a full training step: a batch of tokens, gradients of the hidden states and the head
        dict(name="loss_train_bf16_8192x2048x32000", kind="loss", N=8192, H=2048, V=32000, dtype="bf16", grads="xw",
             mean=True, ignored=True),
        # the loss of a LoRA step: a large vocabulary whose head is frozen
        dict(name="loss_frozen_bf16_4096x2048x131072", kind="loss", N=4096, H=2048, V=131072, dtype="bf16", grads="x",
             mean=True, ignored=False),
        # a policy's loss, each token with a weight of its own: fp32, odd sizes
        dict(name="loss_weighted_fp32_513x1001x50001", kind="loss", N=513, H=1001, V=50001, dtype="fp32", grads="xw",
             mean=False, ignored=True),
        # the score of one token of each of a serving batch
        dict(name="loss_score_bf16_64x4096x32000", kind="loss", N=64, H=4096, V=32000, dtype="bf16", grads="",
             mean=False, ignored=False),
        # the score of one token: what an interactive user waits for
        dict(name="loss_score_bf16_1x2048x131072", kind="loss", N=1, H=2048, V=131072, dtype="bf16", grads="",
             mean=False, ignored=False),
        # a training batch of the benchmark's tokens, few words most of the time
        dict(name="embed_train_bf16_16384x2048_v32000", kind="embed", N=16384, H=2048, V=32000, dtype="bf16", train=True,
             scaled=False, padded=False),
        # a padded batch: fp32, odd sizes
        dict(name="embed_train_fp32_2047x1001_v50001", kind="embed", N=2047, H=1001, V=50001, dtype="fp32", train=True,
             scaled=True, padded=True),
        # one token of each of a serving batch
        dict(name="embed_lookup_bf16_64x4096_v131072", kind="embed", N=64, H=4096, V=131072, dtype="bf16", train=False,
             scaled=True, padded=False),
        # one of a model's weights, once, when it is loaded
        dict(name="quantize_bf16_8192x2048", kind="quantize", N=8192, K=2048, dtype="bf16"),
        # an up projection of a LoRA training step
        dict(name="linear_train_bf16_8192x2048x8192", kind="linear", M=8192, K=2048, N=8192, dtype="bf16", train=True),
        # one token of one sequence
        dict(name="linear_step_bf16_1x2048x8192", kind="linear", M=1, K=2048, N=8192, dtype="bf16", train=False),
        # fp32, odd sizes
        dict(name="linear_train_fp32_1000x1001x4099", kind="linear", M=1000, K=1001, N=4099, dtype="fp32", train=True),
    ]


def _logint(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["loss"] * 4 + ["embed"] * 3 + ["quantize"] + ["linear"] * 3)
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32", "fp16"])
    if kind == "loss":
        grads = rng.choice(["xw", "xw", "x", ""])
        H = rng.choice([2048, 2048, 4096, 1024, 256, 1001, 70])
        V = _logint(rng, 1000, 131072)
        most = min(8192, 8192 * 32000 * 2048 // (V * max(H, 1024) * (4 if dtype == "fp32" else 1)))
        return dict(kind=kind, N=_logint(rng, 1, max(1, most)), H=H, V=V, dtype=dtype, grads=grads,
                    mean=bool(grads) and rng.random() < 0.7, ignored=rng.random() < 0.5)
    if kind == "embed":
        H = rng.choice([2048, 4096, 1024, 256, 1001, 70])
        N, V = _logint(rng, 1, 16384 * 2048 // max(H, 1024)), _logint(rng, 1000, 131072 * 1024 // max(H, 1024))
        return dict(kind=kind, N=N, H=H, V=V, dtype=dtype, train=rng.random() < 0.7, scaled=rng.random() < 0.5,
                    padded=rng.random() < 0.5)
    K, N = rng.choice([2048, 2048, 4096, 8192, 1001, 250]), rng.choice([2048, 8192, 4096, 512, 4099, 97])
    if kind == "quantize":
        return dict(kind=kind, N=_logint(rng, 1, 8192), K=rng.choice([K, _logint(rng, 1, 2048)]), dtype=dtype)
    most = 8192 * 2048 * 8192 // (K * N * (4 if dtype == "fp32" else 2 if dtype == "fp16" else 1))
    return dict(kind=kind, M=_logint(rng, 1, min(8192, most)), K=K, N=N, dtype=dtype, train=rng.random() < 0.6)


# ------------------------------------------------------------------------------------------------ inputs


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))
    rand = lambda *s: torch.randn(*s, device=DEV, generator=gen)  # noqa: E731
    unit = lambda *s: torch.rand(*s, device=DEV, generator=gen)  # noqa: E731
    dtype = DT[c["dtype"]]
    s = {"case": c}
    if c["kind"] == "loss":
        N, H, V = c["N"], c["H"], c["V"]
        w = 3 * H ** -0.5 * rand(V, H)
        target = torch.randint(0, V, (N,), device=DEV, generator=gen)
        at = w[target]  # some tokens are foreseen, some are not
        x = rand(N, H) + 12 * unit(N, 1) * at / at.square().sum(-1, keepdim=True)
        if c["ignored"]:
            target = target.masked_fill(unit(N) < 0.2, -100)
        s.update(x=x.to(dtype), w=w.to(dtype), target=target, weight=rand(N) / N)
        for n in c["grads"]:
            s[n].requires_grad_(True)
    elif c["kind"] == "embed":
        N, H, V = c["N"], c["H"], c["V"]
        ids = (V ** unit(N).double()).long() - 1  # the k-th word about 1 / k times as often as the first
        s["pad"] = V // 2 if c["padded"] else None
        if c["padded"]:
            ids = ids.masked_fill(unit(N) < 1 / 3, s["pad"])
        s.update(ids=ids.clamp(0, V - 1), w=(0.02 * rand(V, H)).to(dtype), scale=H ** 0.5 if c["scaled"] else 1.0)
        if c["train"]:
            s.update(w=s["w"].requires_grad_(True), dy=rand(N, H).to(dtype))
    else:
        w = c["K"] ** -0.5 * rand(c["N"], c["K"]) * (1 + 4 * (unit(c["K"]) < 0.01))  # a few columns stand out
        if c["kind"] == "quantize":
            s.update(w=w.to(dtype))
            return s
        codes, scales = _plain_quantize(w)
        s.update(codes=codes, scales=scales, x=rand(c["M"], c["K"]).to(dtype))
        if c["train"]:
            s.update(x=s["x"].requires_grad_(True), dy=rand(c["M"], c["N"]).to(dtype))
    return s


# ------------------------------------------------------------------------------------------------ plain forms


def _plain_quantize(w):
    """Codes [N, K / 2] (two to a byte, the even element low) and scales [N, K / 32] (biased exponents), K padded to
    blocks of 32 with zeros."""
    w = torch.nn.functional.pad(w.float(), (0, -w.shape[1] % 32)).unflatten(-1, (-1, 32))
    e = torch.frexp(w.abs().amax(-1)).exponent - 1 - 2  # the largest element in [4, 8)
    e = e.clamp_min(-127).masked_fill((w == 0).all(-1), -127)
    m = torch.ldexp(w.abs().double(), -e[..., None]).float()
    step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0))
    q = (torch.round(m / step) * step).clamp_max(6.0)
    code = torch.where(q < 2, 2 * q, torch.where(q < 4, q + 2, q / 2 + 4)).to(torch.uint8) | (torch.signbit(w) * 8).to(torch.uint8)
    code = code.flatten(-2)
    return code[:, 0::2] | code[:, 1::2] << 4, (e + 127).to(torch.uint8)


def _plain_values(codes, scales, K):
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    q = (code & 7).float()
    q = torch.where(q < 4, q / 2, torch.where(q < 6, q - 2, 2 * q - 8))
    q = torch.where(code > 7, -q, q).unflatten(-1, (-1, 32))
    return torch.ldexp(q, scales.int()[..., None] - 127).flatten(-2)[:, :K]


def run(state):
    s, c = state, state["case"]
    if own:
        return _run_own(s, c)
    kind = c["kind"]
    if kind == "loss":
        x, w = s["x"].detach().float(), s["w"].detach().float()
        z = x @ w.t()
        top = z.max(-1, keepdim=True).values
        e = (z - top).exp()
        total = e.sum(-1, keepdim=True)
        live = s["target"] != -100
        at = s["target"].clamp_min(0)[:, None]
        loss = (total.log() + top - z.gather(-1, at))[:, 0].masked_fill(~live, 0.0)
        count = live.sum().clamp_min(1)
        out = {"loss": loss.sum() / count if c["mean"] else loss}
        if c["grads"]:
            d = live / count if c["mean"] else s["weight"] * live
            dz = e / total
            dz.scatter_add_(-1, at, torch.full_like(top, -1.0))
            dz *= d[:, None]
            out["dx"] = (dz @ w).to(s["x"].dtype)
            if "w" in c["grads"]:
                out["dw"] = (dz.t() @ x).to(s["w"].dtype)
        return out
    if kind == "embed":
        w = s["w"].detach()
        out = {"y": (w[s["ids"]].float() * s["scale"]).to(w.dtype)}
        if c["train"]:
            dy = s["dy"].double()
            if c["padded"]:
                dy = dy * (s["ids"] != s["pad"])[:, None]
            dw = torch.zeros(w.shape, device=w.device, dtype=torch.float64).index_add_(0, s["ids"], dy)
            out["dw"] = (dw * s["scale"]).to(w.dtype)
        return out
    if kind == "quantize":
        return {"values": _plain_values(*_plain_quantize(s["w"]), c["K"]).to(s["w"].dtype)}
    w = _plain_values(s["codes"], s["scales"], c["K"])
    out = {"y": (s["x"].detach().float() @ w.t()).to(s["x"].dtype)}
    if c["train"]:
        out["dx"] = (s["dy"].float() @ w).to(s["x"].dtype)
    return out


# ------------------------------------------------------------------------------------------------ the framework's calls


def _run_own(s, c):
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    kind = c["kind"]
    if kind == "loss":
        from linear_loss import linear_cross_entropy
        loss = linear_cross_entropy(s["x"], s["w"], s["target"], reduction="mean" if c["mean"] else "none")
        out = {"loss": loss}
        if c["grads"]:
            grads = torch.autograd.grad(loss, [s[n] for n in c["grads"]], None if c["mean"] else s["weight"])
            out.update(zip(["d" + n for n in c["grads"]], grads))
        return out
    if kind == "embed":
        from embedding import embedding
        y = embedding(s["ids"], s["w"], scale=s["scale"], padding_idx=s["pad"])
        out = {"y": y}
        if c["train"]:
            out["dw"] = torch.autograd.grad(y, s["w"], s["dy"])[0]
        return out
    import mxfp4
    if kind == "quantize":
        return {"values": mxfp4.dequantize(mxfp4.quantize(s["w"]), s["w"].dtype)}
    y = mxfp4.linear(s["x"], mxfp4.Weight(s["codes"], s["scales"], c["K"]))
    out = {"y": y}
    if c["train"]:
        out["dx"] = torch.autograd.grad(y, s["x"], s["dy"])[0]
    return out


# ------------------------------------------------------------------------------------------------ work


def work(case):
    c = case
    e = SIZE[c["dtype"]]
    if c["kind"] == "loss":
        x, w, n = c["N"] * c["H"] * e, c["V"] * c["H"] * e, 2 * c["N"] * c["V"] * c["H"]
        out = (x if "x" in c["grads"] else 0) + (w if "w" in c["grads"] else 0)
        return {"bytes": x + w + out + c["N"] * 12, "flops": n * (1 + len(c["grads"]))}
    if c["kind"] == "embed":
        rows = c["N"] * c["H"]
        n = 2 * rows * e + 8 * c["N"]
        return {"bytes": n + (rows + c["V"] * c["H"]) * e if c["train"] else n, "flops": rows * (2 if c["train"] else 1)}
    n = c["N"] * c["K"]
    if c["kind"] == "quantize":
        return {"bytes": 2 * n * e + n * 17 // 32, "flops": 4 * n}
    both = 2 if c["train"] else 1
    return {"bytes": n * 17 // 32 + both * c["M"] * (c["K"] + c["N"]) * e, "flops": both * 2 * c["M"] * n}


# ------------------------------------------------------------------------------------------------ 64 bits


_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def exact(case, seed):
    c, s = case, prepare(case, seed)
    kind = c["kind"]
    table = torch.tensor(_E2M1, device=DEV, dtype=torch.float64)
    if kind == "loss":
        x, w, N = s["x"].detach().double(), s["w"].detach().double(), c["N"]
        live = s["target"] >= 0
        d = (live.double() / max(1, int(live.sum())) if c["mean"] else s["weight"].double() * live)
        loss, dx, dw = [], torch.empty_like(x), torch.zeros_like(w) if "w" in c["grads"] else None
        for i in range(0, N, 1024):  # rows at a time
            part = slice(i, min(N, i + 1024))
            logp = torch.log_softmax(x[part] @ w.t(), -1)
            rows, at = torch.arange(logp.shape[0], device=DEV), torch.where(live[part], s["target"][part], 0)
            loss.append(torch.where(live[part], -logp[rows, at], 0.0))
            if c["grads"]:
                dz = logp.exp_()
                dz[rows, at] -= 1
                dz *= d[part, None]
                dx[part] = dz @ w
                if dw is not None:
                    dw += dz.t().contiguous() @ x[part]
        loss = torch.cat(loss)
        out = {"loss": loss.sum() / max(1, int(live.sum())) if c["mean"] else loss}
        if c["grads"]:
            out["dx"] = dx
            if dw is not None:
                out["dw"] = dw
        return out
    if kind == "embed":
        out = {"y": torch.index_select(s["w"].detach().double(), 0, s["ids"]) * s["scale"]}
        if c["train"]:
            order = torch.argsort(s["ids"], stable=True)
            sums = torch.cumsum(s["dy"].double()[order], 0)
            words, counts = torch.unique_consecutive(s["ids"][order], return_counts=True)
            last = sums[torch.cumsum(counts, 0) - 1]
            dw = torch.zeros(c["V"], c["H"], device=DEV, dtype=torch.float64)
            dw[words] = torch.diff(last, dim=0, prepend=torch.zeros_like(last[:1])) * s["scale"]
            if c["padded"]:
                dw[s["pad"]] = 0
            out["dw"] = dw
        return out
    if kind == "quantize":
        w = torch.nn.functional.pad(s["w"].double(), (0, -c["K"] % 32)).unflatten(-1, (-1, 32))
        most = w.abs().amax(-1, keepdim=True)
        unit = torch.where(most > 0, torch.exp2(torch.floor(torch.log2(most)) - 2), torch.ones_like(most))
        m = w.abs() / unit
        up = torch.bucketize(m, (table[1:] + table[:-1]) / 2, right=False)  # of two as near the lower one
        tie = m == torch.cat([(table[1:] + table[:-1]) / 2, table[-1:] * 2])[up]
        return {"values": (table[up + (tie & (up % 2 == 1))] * unit * torch.sign(w)).flatten(-2)[:, :c["K"]]}
    code = torch.stack([s["codes"] % 16, s["codes"] // 16], -1).flatten(-2).long()
    w = table[code % 8] * torch.where(code >= 8, -1.0, 1.0)
    w = (w.unflatten(-1, (-1, 32)) * torch.exp2(s["scales"].double() - 127)[..., None]).flatten(-2)[:, :c["K"]]
    out = {"y": s["x"].detach().double() @ w.t()}
    if c["train"]:
        out["dx"] = s["dy"].double() @ w
    return out
