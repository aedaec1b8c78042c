"""Log probabilities of given tokens from a model's logits, with the entropy of each distribution and its top
alternatives, and the gradient of the logits: the loss of a training step, the score of sampled text.  The reference
takes its loss in slices to keep a full softmax out of memory (``tools/ft_lowmem_loss.py:31-71``); here no probability
is ever stored: one read of the logits forward, one read and the write of their gradient backward.  Tensors must live on
a ROCm device; there is no CPU path.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

import gdn_lib as L

Array = torch.Tensor


class TokenLogprobs(NamedTuple):
    logp: Array                  # [...] float32
    entropy: Optional[Array]     # [...] float32, with entropy=True
    top_ids: Optional[Array]     # [..., top] int64
    top_logp: Optional[Array]    # [..., top] float32, not differentiable


def _rows(z: Array) -> tuple[Array, tuple[int, int, int, int]]:
    """The logits as [outer][inner] rows: (tensor, (outer, inner, stride_outer, stride_inner)); copied only where its
    rows are not contiguous or do not lie on two strides."""
    V = z.shape[-1]
    if z.stride(-1) != 1 and V > 1:
        z = z.contiguous()
    lead = [(n, s) for n, s in zip(z.shape[:-1], z.stride()[:-1]) if n != 1]
    merged: list[tuple[int, int]] = []
    for n, s in lead:
        if merged and merged[-1][1] == n * s:
            merged[-1] = (merged[-1][0] * n, s)
        else:
            merged.append((n, s))
    if len(merged) > 2:
        z = z.contiguous()
        merged = [(z.numel() // V, V)]
    while len(merged) < 2:
        merged.insert(0, (1, 0))
    (o, so), (i, si) = merged
    return z, (o, i, so, si)


def _forward(z, layout, targets, entropy, top, ignore_index, need_grad):
    """(logp, entropy, ids, top_logp), and the rows' statistics for the backward."""
    dev, lead, V = z.device, z.shape[:-1], z.shape[-1]
    rows = targets.numel()
    f32 = dict(dtype=torch.float32, device=dev)
    logp = torch.empty(lead, **f32)
    ent = torch.empty(lead, **f32) if entropy else None
    stat = torch.empty((rows, 2), **f32) if need_grad else None
    ids = torch.empty((*lead, top), dtype=torch.int64, device=dev) if top else None
    tlp = torch.empty((*lead, top), **f32) if top else None
    lib = L.load()
    nws = lib.gdn_logprobs_workspace_bytes(rows, V, top)
    ws = torch.empty((nws,), dtype=torch.uint8, device=dev)
    outer, inner, so, si = layout
    with L.on_device(dev):
        L.check(lib.gdn_logprobs_fwd(z.data_ptr(), targets.data_ptr(), logp.data_ptr(), L.ptr(ent), L.ptr(stat),
                                     L.ptr(ids), L.ptr(tlp), ws.data_ptr(), nws, outer, inner, V, so, si,
                                     ignore_index, top, L.DTYPE_CODE[z.dtype], L.stream_handle(dev)))
    return (logp, ent, ids, tlp), stat


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, layout, targets, entropy, top, ignore_index):
        ctx.set_materialize_grads(False)
        out, stat = _forward(z, layout, targets, entropy, top, ignore_index, True)
        ctx.save_for_backward(z, targets, stat, out[1])
        ctx.meta = (*layout, ignore_index, z.shape)
        ctx.mark_non_differentiable(*[t for t in out[2:] if t is not None])
        return out

    @staticmethod
    def backward(ctx, dlogp, dent, _ids, _tlp):
        z, targets, stat, ent = ctx.saved_tensors
        outer, inner, so, si, ignore_index, shape = ctx.meta
        dev = z.device
        if dlogp is None and dent is None:
            return (None,) * 6
        dlogp = None if dlogp is None else dlogp.float().contiguous()
        dent = None if dent is None else dent.float().contiguous()
        dz = torch.empty(shape, dtype=z.dtype, device=dev)
        with L.on_device(dev):
            L.check(L.load().gdn_logprobs_bwd(z.data_ptr(), targets.data_ptr(), stat.data_ptr(), L.ptr(ent),
                                              L.ptr(dlogp), L.ptr(dent), dz.data_ptr(), outer, inner, shape[-1], so, si,
                                              ignore_index, L.DTYPE_CODE[z.dtype], L.stream_handle(dev)))
        return (*L.once((z, dlogp, dent), dz), None, None, None, None, None)


def token_logprobs(logits: Array, targets: Array, *, entropy: bool = False, top: int = 0,
                   ignore_index: int = -100) -> TokenLogprobs:
    """Log probabilities of ``targets`` [...] under softmax(``logits`` [..., V]).

    ``logp`` is 0, without a gradient, where ``targets == ignore_index``, and NaN where a target lies outside [0, V).
    ``entropy`` adds the entropy of every row (nats), ``top`` the ``top`` most likely tokens and their log
    probabilities, equal ones in the order of their ids (at most 64).  Differentiable in the logits through ``logp`` and
    ``entropy``.  Logits of -inf (banned tokens) have probability 0; a row of nothing else has log probabilities -inf,
    entropy 0 and no gradient.  Logits may be a view with two row strides (``logits[:, :-1]``): it is not copied."""
    if logits.dim() < 1 or tuple(targets.shape) != tuple(logits.shape[:-1]):
        raise ValueError(f"targets must have the logits' leading shape; got {tuple(targets.shape)} for "
                         f"{tuple(logits.shape)}")
    if logits.dtype not in L.DTYPE_CODE:
        raise ValueError(f"unsupported dtype {logits.dtype}; use float32, bfloat16 or float16")
    if targets.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"targets must be int64 or int32; got {targets.dtype}")
    if logits.shape[-1] == 0 or not 0 <= top <= logits.shape[-1]:
        raise ValueError(f"top must be between 0 and V = {logits.shape[-1]}, V positive; got {top}")
    if logits.device.type != "cuda":
        raise RuntimeError("token_logprobs runs on a ROCm GPU only; got tensors on " + str(logits.device))
    if targets.device != logits.device:
        raise ValueError("all inputs must be on the same device")
    args = (*_rows(logits), targets.to(torch.int64).contiguous(), bool(entropy), int(top), int(ignore_index))
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenLogprobs(*_TokenLogprobs.apply(*args))
    return TokenLogprobs(*_forward(*args, False)[0])
