"""The loss of a language model from its last hidden states and its head, without the logits: cross entropy of x W^T, with the
gradients of both.  The reference takes its loss in slices to keep the logits out of memory
(``tools/ft_lowmem_loss.py:31-71``); here a slice of them exists in registers only, and in the backward pass as one piece of
probabilities at a time.  ``token_logprobs`` is the same loss of logits that exist.  Tensors must live on a ROCm device; there
is no CPU path.
"""

from __future__ import annotations

import torch

import gdn_lib as L

Array = torch.Tensor
REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def _rows(t: Array) -> Array:
    """[..., H] as rows with contiguous channels, copied only where it has to be."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if t.stride(1) != 1 and t.shape[1] > 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        t = t.contiguous()
    return t


def _forward(x, w, targets, ignore_index, reduction, need_grad):
    """(losses [N], their total and its factor, the tokens' statistics; None where not asked for)"""
    dev = x.device
    (N, H), V = x.shape, w.shape[0]
    lib, dtype = L.load(), L.DTYPE_CODE[x.dtype]
    loss = torch.empty((N,), dtype=torch.float32, device=dev)
    stat = torch.empty((N + 1, 2), dtype=torch.float32, device=dev) if need_grad else None
    total = torch.empty((), dtype=torch.float32, device=dev) if reduction else None
    factor = torch.empty((), dtype=torch.float32, device=dev) if reduction else None
    nws = lib.gdn_linear_loss_workspace_bytes(N, H, V, dtype, L.rows_lie_well(x, w), 0, 0)
    ws = torch.empty((nws,), dtype=torch.uint8, device=dev)
    with L.on_device(dev):
        L.check(lib.gdn_linear_loss_fwd(x.data_ptr(), w.data_ptr(), targets.data_ptr(), loss.data_ptr(), L.ptr(stat),
                                        L.ptr(total), L.ptr(factor), ws.data_ptr(), nws, N, H, V, L.row_stride(x), L.row_stride(w),
                                        ignore_index, reduction, dtype, L.stream_handle(dev)))
    return loss, total, factor, stat


class _LinearLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, targets, ignore_index, reduction):
        loss, total, factor, stat = _forward(x, w, targets, ignore_index, reduction, True)
        ctx.save_for_backward(x, w, targets, stat, factor)
        ctx.meta = (ignore_index, reduction)
        return total if reduction else loss

    @staticmethod
    def backward(ctx, dloss):
        x, w, targets, stat, factor = ctx.saved_tensors
        ignore_index, reduction = ctx.meta
        dev, (N, H), V = x.device, x.shape, w.shape[0]
        need_x, need_w = ctx.needs_input_grad[:2]
        dloss = dloss.float().contiguous()
        if N == 0:
            dx = torch.empty_like(x) if need_x else None
            dw = w.new_zeros(w.shape) if need_w else None
            return (*L.once((x, w, dloss), dx, dw), None, None, None)
        dx = torch.empty((N, H), dtype=x.dtype, device=dev) if need_x else None
        dw = torch.empty((V, H), dtype=w.dtype, device=dev) if need_w else None
        lib, dtype = L.load(), L.DTYPE_CODE[x.dtype]
        nws = lib.gdn_linear_loss_workspace_bytes(N, H, V, dtype, L.rows_lie_well(x, w), need_x, need_w)
        ws = torch.empty((nws,), dtype=torch.uint8, device=dev)
        with L.on_device(dev):
            L.check(lib.gdn_linear_loss_bwd(x.data_ptr(), w.data_ptr(), targets.data_ptr(), stat.data_ptr(), dloss.data_ptr(),
                                            0 if reduction else 1, L.ptr(factor), L.ptr(dx), L.ptr(dw),
                                            ws.data_ptr(), nws, N, H, V, L.row_stride(x), L.row_stride(w), ignore_index,
                                            dtype, L.stream_handle(dev)))
        return (*L.once((x, w, dloss), dx, dw), None, None, None)


def linear_cross_entropy(x: Array, weight: Array, targets: Array, *, ignore_index: int = -100,
                         reduction: str = "mean") -> Array:
    """Cross entropy (nats, float32) of the logits ``x`` [..., H] @ ``weight`` [V, H]^T at ``targets`` [...].

    ``reduction`` "none" gives the loss of every token, "sum" their sum, "mean" their mean over the tokens that count: those
    whose target is not ``ignore_index`` (0 if none does).  An ignored token has loss 0 and no gradient, whatever ``x`` holds
    there; a target outside [0, V) makes the token's loss NaN, and the gradients that it enters.  Differentiable in ``x`` and
    ``weight``; a frozen weight costs no gradient of its own.  ``x`` and ``weight`` may be views with contiguous channels.

    Tokens that do not count cost no time where there are many (2048 and more in all).  At most 2^20 tokens.

    Memory beside the gradients.  Words come in pieces of 2^26 probabilities over all tokens, or of 256 words if that is more.
    Forward: 8 bytes for each token and 64 words, up to 512 MB, and copies of what the matrix products cannot read as it lies:
    ``x`` from 2048 tokens on, and of float32, odd sizes and rows off 16 bytes or more than 8 MiB apart ``x`` and a piece of
    ``weight``, 2 bytes an element (float32 4, or 6 up to 128 tokens).  Backward: these copies (float32 6 bytes), a piece's
    probabilities at 4 bytes each (up to 128 float32 tokens 6); for ``x``'s gradient float32 sums of its size, of few tokens
    in up to 32 parts; for ``weight``'s another copy of ``x`` and, of few words, float32 sums of a piece in up to 8 parts.

    bfloat16 and float16 inputs enter with all their bits, and gradients are as good as 32-bit sums rounded once (float16, whose
    gradients end at 2^-25, as long as cotangents times ``x`` stay below 2^15: probabilities are kept to 2^-40).  float32
    inputs are sums of 16-bit terms, which hold no infinities: those may count as NaN.  Up to 128 tokens the terms are exact.
    With more they leave out 2^-22 of a number, or 2^-39 of the largest of its token (``x``, in the loss and its own gradient), of
    ``weight``, or of ``x`` (in ``weight``'s gradient), whichever is more, and gradients 2^-22 of a probability or 2^-51."""
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x must be [..., H] and weight [V, H]; got {tuple(x.shape)} and {tuple(weight.shape)}")
    if tuple(targets.shape) != tuple(x.shape[:-1]):
        raise ValueError(f"targets must have x's leading shape; got {tuple(targets.shape)} for {tuple(x.shape)}")
    if x.dtype not in L.DTYPE_CODE or weight.dtype != x.dtype:
        raise ValueError(f"x and weight must both be float32, bfloat16 or float16; got {x.dtype} and {weight.dtype}")
    if targets.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"targets must be int64 or int32; got {targets.dtype}")
    if weight.numel() == 0:
        raise ValueError("weight must not be empty")
    if reduction not in REDUCTIONS:
        raise ValueError(f"reduction must be one of {', '.join(REDUCTIONS)}; got {reduction!r}")
    L.refuse_tangents("linear_cross_entropy", x, weight)
    if x.device.type != "cuda":
        raise RuntimeError("linear_cross_entropy runs on a ROCm GPU only; got tensors on " + str(x.device))
    if weight.device != x.device or targets.device != x.device:
        raise ValueError("all inputs must be on the same device")
    flat = targets.to(torch.int64).reshape(-1).contiguous()
    code = REDUCTIONS[reduction]
    lead, x, weight = x.shape[:-1], _rows(x), _rows(weight)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        out = _LinearLoss.apply(x, weight, flat, int(ignore_index), code)
    else:
        loss, total, _, _ = _forward(x, weight, flat, int(ignore_index), code, False)
        out = total if code else loss
    return out if code else out.view(lead)
