"""Rotary positions: pairs of channels of q and k turned by angles that grow with their token's position, so that their
products depend on distances.  One HIP kernel for q and k, forward and backward; angles are formed in 64 bits, so far
positions keep their accuracy.  Tensors must live on a ROCm device; there is no CPU path.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

import gdn_lib as L

Array = torch.Tensor


def rotary_frequencies(dim: int, base: float = 10000.0, *, scaling: Optional[str] = None, factor: float = 1.0,
                       trained_length: int = 4096, fast_turns: float = 32.0, slow_turns: float = 1.0,
                       device=None) -> tuple[Array, float]:
    """(inverse frequencies [dim / 2] in float64, the factor on the rotated values) for ``rotary``.

    ``scaling`` stretches positions beyond the trained length by ``factor``:
      None      none: base^(-2i / dim), factor 1
      "linear"  every frequency divided by ``factor``
      "base"    the base raised so that the slowest pair is slowed by ``factor`` and the fastest not at all
      "parts"   pairs with more than ``fast_turns`` turns over ``trained_length`` kept, those with fewer than
                ``slow_turns`` divided by ``factor``, a linear blend in the turns between; the rotated values grow by
                0.1 ln(factor) + 1 (so that the softmax or the state keeps its temperature)
    """
    if dim <= 0 or dim % 2:
        raise ValueError(f"the rotated part must be even and positive; got {dim}")
    if not base > 0 or not factor >= 1.0:
        raise ValueError("base must be positive and factor at least 1")
    steps = torch.arange(0, dim, 2, dtype=torch.float64, device=device) / dim
    if scaling == "base":
        base = base * factor ** (dim / max(dim - 2, 1))
    inv = base ** -steps
    if scaling in (None, "base"):
        return inv, 1.0
    if scaling == "linear":
        return inv / factor, 1.0
    if scaling != "parts":
        raise ValueError(f"scaling must be None, 'linear', 'base' or 'parts'; got {scaling!r}")
    if not fast_turns > slow_turns:
        raise ValueError("fast_turns must be greater than slow_turns")
    turns = trained_length * inv / (2 * math.pi)
    keep = ((turns - slow_turns) / (fast_turns - slow_turns)).clamp(0, 1)
    return inv / factor * (1 - keep) + inv * keep, 0.1 * math.log(factor) + 1.0


def _launch(q: Array, k: Array, pos: Array, inv: Array, interleaved: bool, factor: float, backward: bool):
    B, T, Hq, D = q.shape
    Hk = k.shape[2]
    dev = q.device
    q = q if q.stride(-1) == 1 or D == 1 else q.contiguous()
    k = k if k.stride(-1) == 1 or D == 1 else k.contiguous()
    qo = torch.empty((B, T, Hq, D), dtype=q.dtype, device=dev)
    ko = torch.empty((B, T, Hk, D), dtype=k.dtype, device=dev)
    pb = pos.stride(0) if pos.dim() == 2 else 0
    with L.on_device(dev):
        L.check(L.load().gdn_rotary(q.data_ptr(), k.data_ptr(), qo.data_ptr(), ko.data_ptr(), pos.data_ptr(),
                                    inv.data_ptr(), *q.stride()[:3], *k.stride()[:3], pb, pos.stride(-1), B, T, Hq, Hk,
                                    D, 2 * inv.numel(), int(interleaved), int(backward),
                                    int(pos.dtype == torch.int64), factor, L.DTYPE_CODE[q.dtype],
                                    L.stream_handle(dev)))
    return qo, ko


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, pos, inv, interleaved, factor):
        ctx.save_for_backward(pos, inv)
        ctx.meta = (interleaved, factor)
        return _launch(q, k, pos, inv, interleaved, factor, False)

    @staticmethod
    def backward(ctx, dq, dk):
        pos, inv = ctx.saved_tensors
        return (*L.once((dq, dk), *_launch(dq, dk, pos, inv, *ctx.meta, True)), None, None, None, None)


def rotary(q: Array, k: Array, positions: Array, inv_freq: Array, *, interleaved: bool = False,
           factor: float = 1.0) -> tuple[Array, Array]:
    """q [B, T, Hq, D] and k [B, T, Hk, D] with pair i of each head's first R = 2 len(inv_freq) channels turned by
    ``positions * inv_freq[i]`` and multiplied by ``factor``; channels from R on pass through.  Pairs are (i, i + R/2),
    or (2i, 2i + 1) with ``interleaved``.  ``positions`` [T] or [B, T] are int64 or int32, ``inv_freq`` and ``factor``
    as ``rotary_frequencies`` returns them (float64; float32 is widened).  q and k may be strided views; the outputs are
    contiguous and have their type.  Differentiable in q and k."""
    if q.dim() != 4 or k.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError(f"rotary expects q [B, T, Hq, D] and k [B, T, Hk, D]; got {tuple(q.shape)}, {tuple(k.shape)}")
    B, T, _, D = q.shape
    if q.dtype != k.dtype or q.dtype not in L.DTYPE_CODE:
        raise ValueError(f"q and k must share one of float32, bfloat16, float16; got {q.dtype}, {k.dtype}")
    if tuple(positions.shape) not in ((T,), (B, T)):
        raise ValueError(f"positions must be [T] or [B, T] = {(B, T)}; got {tuple(positions.shape)}")
    if positions.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"positions must be int64 or int32; got {positions.dtype}")
    if inv_freq.dim() != 1 or not 0 < 2 * inv_freq.numel() <= D:
        raise ValueError(f"inv_freq must hold between 1 and D / 2 = {D // 2} frequencies; got {tuple(inv_freq.shape)}")
    L.refuse_tangents("rotary", q, k)
    if q.device.type != "cuda":
        raise RuntimeError("rotary runs on a ROCm GPU only; got tensors on " + str(q.device))
    if any(t.device != q.device for t in (k, positions, inv_freq)):
        raise ValueError("all inputs must be on the same device")
    inv = inv_freq.detach().to(torch.float64).contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad):
        return _Rotary.apply(q, k, positions, inv, bool(interleaved), float(factor))
    return _launch(q, k, positions, inv, bool(interleaved), float(factor), False)
