"""Rows of an embedding table, scaled, and the table's gradient by sorted tokens: the first operator of a language model,
whose backward pass torch leaves to sums in an order of arrival.  Tensors must live on a ROCm device; there is no CPU path
(``Embedding``, an ``nn.Embedding`` that calls it, keeps torch's own there).
"""

from __future__ import annotations

from typing import Optional

import torch

import gdn_lib as L

Array = torch.Tensor


def _forward(ids, w, scale):
    y = torch.empty((*ids.shape, w.shape[1]), dtype=w.dtype, device=w.device)
    with L.on_device(w.device):
        L.check(L.load().gdn_embedding_fwd(ids.data_ptr(), w.data_ptr(), y.data_ptr(), ids.numel(), *w.shape, w.stride(0), scale,
                                           L.DTYPE_CODE[w.dtype], L.stream_handle(w.device)))
    return y


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, w, ids, scale, padding_idx):
        ctx.save_for_backward(ids)
        ctx.meta = (w.shape, scale, padding_idx)
        return _forward(ids, w, scale)

    @staticmethod
    def backward(ctx, dy):
        ids, = ctx.saved_tensors
        (V, H), scale, padding_idx = ctx.meta
        N, dev = ids.numel(), dy.device
        rows = dy if dy.dim() == 2 else dy.reshape(N, H)
        if rows.stride(1) != 1:
            rows = rows.contiguous()
        dw = torch.empty((V, H), dtype=dy.dtype, device=dev)
        lib = L.load()
        nws = lib.gdn_embedding_bwd_workspace_bytes(N, V, H)
        ws = torch.empty((nws,), dtype=torch.uint8, device=dev)
        with L.on_device(dev):
            L.check(lib.gdn_embedding_bwd(ids.data_ptr(), rows.data_ptr(), dw.data_ptr(), ws.data_ptr(), nws, N, V, H,
                                          rows.stride(0), -1 if padding_idx is None else padding_idx, scale,
                                          L.DTYPE_CODE[dy.dtype], L.stream_handle(dev)))
        return (*L.once((dy,), dw), None, None, None)


def embedding(ids: Array, weight: Array, *, scale: float = 1.0, padding_idx: Optional[int] = None) -> Array:
    """``scale * weight[ids]`` for ``ids`` [...] (int64 or int32) and ``weight`` [V, H]: [..., H] of the weight's type.

    Differentiable in ``weight``: its gradient is summed in 64 bits, 32 tokens of a word at a time in their order, and rounded
    to 32 bits and its type, the same bits every time.  The backward pass takes half a byte of workspace for each element of the
    output and 16 bytes for each token.  Tokens equal to ``padding_idx`` have no gradient.  An id outside [0, V) gives a row of
    NaN, without a gradient.  ``weight`` may be a view with contiguous rows."""
    if weight.dim() != 2 or weight.numel() == 0:
        raise ValueError(f"weight must be [V, H] and not empty; got {tuple(weight.shape)}")
    if weight.dtype not in L.DTYPE_CODE:
        raise ValueError(f"unsupported dtype {weight.dtype}; use float32, bfloat16 or float16")
    if ids.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"ids must be int64 or int32; got {ids.dtype}")
    if padding_idx is not None and not 0 <= padding_idx < weight.shape[0]:
        raise ValueError(f"padding_idx must be in [0, {weight.shape[0]}); got {padding_idx}")
    L.refuse_tangents("embedding", weight)
    if weight.device.type != "cuda":
        raise RuntimeError("embedding runs on a ROCm GPU only; got tensors on " + str(weight.device))
    if ids.device != weight.device:
        raise ValueError("all inputs must be on the same device")
    if weight.stride(1) != 1 or weight.stride(0) < 0:
        weight = weight.contiguous()
    ids = ids.to(torch.int64).contiguous()
    if torch.is_grad_enabled() and weight.requires_grad:
        return _Embedding.apply(weight, ids, float(scale), padding_idx)
    return _forward(ids, weight, float(scale))


class Embedding(torch.nn.Embedding):
    """``nn.Embedding`` (its parameters, its state) through ``embedding``, with a factor on the rows.  On the CPU it is torch's
    own, scaled."""

    def __init__(self, num_embeddings: int, embedding_dim: int, padding_idx: Optional[int] = None, *, scale: float = 1.0, **kw):
        super().__init__(num_embeddings, embedding_dim, padding_idx, **kw)
        if self.max_norm is not None or self.scale_grad_by_freq or self.sparse:
            raise ValueError("max_norm, scale_grad_by_freq and sparse are not supported")
        self.scale = scale

    def forward(self, ids: Array) -> Array:
        if self.weight.device.type == "cuda":
            return embedding(ids, self.weight, scale=self.scale, padding_idx=self.padding_idx)
        y = super().forward(ids)
        return y if self.scale == 1.0 else (y.double() * self.scale).to(y.dtype)
