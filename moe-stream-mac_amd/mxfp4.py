"""Frozen weights in microscaled 4-bit floating point (MXFP4: blocks of 32 elements with a common power of two), and products
with them: the base weights under LoRA adapters, which the reference keeps in 4 bits as well (MLX's affine format), here in the
format of the card's own 4-bit types.  17 / 32 of a byte for each element; the gradient of the input, none of the weight.
Tensors must live on a ROCm device; there is no CPU path.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

import gdn_lib as L

Array = torch.Tensor
BLOCK = 32


class Weight(NamedTuple):
    """A weight [N, K]: ``codes`` [N, ceil(K / 32) * 16] uint8, two elements (sign, e2m1) to a byte, the even one low;
    ``scales`` [N, ceil(K / 32)] uint8, the biased exponents of the blocks' powers of two (255: NaN); ``columns`` = K."""
    codes: Array
    scales: Array
    columns: int

    @property
    def shape(self) -> tuple[int, int]:
        return self.codes.shape[0], self.columns


def _check(q: Weight) -> None:
    codes, scales, K = q
    blocks = -(-K // BLOCK)
    if K <= 0 or codes.dim() != 2 or codes.shape[1] != blocks * 16 or tuple(scales.shape) != (codes.shape[0], blocks):
        raise ValueError(f"codes must be [N, {blocks * 16}] and scales [N, {blocks}] for {K} columns; got {tuple(codes.shape)} "
                         f"and {tuple(scales.shape)}")
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise ValueError(f"codes and scales must be uint8; got {codes.dtype} and {scales.dtype}")
    if not codes.is_contiguous() or not scales.is_contiguous():
        raise ValueError("codes and scales must be contiguous")
    if scales.device != codes.device:
        raise ValueError("codes and scales must be on the same device")


def _on_gpu(t: Array, what: str) -> None:
    if t.device.type != "cuda":
        raise RuntimeError(f"{what} runs on a ROCm GPU only; got tensors on {t.device}")


def quantize(w: Array) -> Weight:
    """``w`` [N, K] in blocks of 32 along K.  A block's power of two takes its largest magnitude to [4, 8); elements round to the
    nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6, ties to the even code.  A block with an infinite or NaN element becomes NaN."""
    if w.dim() != 2 or w.shape[1] == 0:
        raise ValueError(f"w must be [N, K]; got {tuple(w.shape)}")
    if w.dtype not in L.DTYPE_CODE:
        raise ValueError(f"unsupported dtype {w.dtype}; use float32, bfloat16 or float16")
    _on_gpu(w, "quantize")
    w = w.detach()
    if w.stride(1) != 1 and w.shape[1] > 1:
        w = w.contiguous()
    N, K = w.shape
    blocks = -(-K // BLOCK)
    codes = torch.empty((N, blocks * 16), dtype=torch.uint8, device=w.device)
    scales = torch.empty((N, blocks), dtype=torch.uint8, device=w.device)
    with L.on_device(w.device):
        L.check(L.load().gdn_mxfp4_quantize(w.data_ptr(), codes.data_ptr(), scales.data_ptr(), N, K, w.stride(0),
                                            L.DTYPE_CODE[w.dtype], L.stream_handle(w.device)))
    return Weight(codes, scales, K)


def dequantize(q: Weight, dtype: torch.dtype = torch.bfloat16) -> Array:
    """The values [N, K]: exact in float32 and bfloat16, rounded in float16."""
    _check(q)
    if dtype not in L.DTYPE_CODE:
        raise ValueError(f"unsupported dtype {dtype}; use float32, bfloat16 or float16")
    _on_gpu(q.codes, "dequantize")
    dev = q.codes.device
    out = torch.empty(q.shape, dtype=dtype, device=dev)
    with L.on_device(dev):
        L.check(L.load().gdn_mxfp4_dequantize(q.codes.data_ptr(), q.scales.data_ptr(), out.data_ptr(), *out.shape,
                                              L.DTYPE_CODE[dtype], L.stream_handle(dev)))
    return out


def _product(name: str, x: Array, q: Weight, backward: bool) -> Array:
    """Rows of x times the weight's transpose, or with backward times the weight."""
    N, K = q.shape
    M, dev = x.shape[0], x.device
    if M > 1 and x.stride(0) < x.shape[1] or x.stride(1) != 1 and x.shape[1] > 1:
        x = x.contiguous()
    y = torch.empty((M, K if backward else N), dtype=x.dtype, device=dev)
    lib, dtype = L.load(), L.DTYPE_CODE[x.dtype]
    nws = lib.gdn_mxfp4_linear_workspace_bytes(M, K, N, dtype, L.rows_lie_well(x), backward)
    ws = torch.empty((nws,), dtype=torch.uint8, device=dev) if nws else None
    with L.on_device(dev):
        L.check(getattr(lib, name)(x.data_ptr(), q.codes.data_ptr(), q.scales.data_ptr(), y.data_ptr(), L.ptr(ws), nws, M, K, N,
                                   L.row_stride(x), dtype, L.stream_handle(dev)))
    return y


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, codes, scales, K):
        ctx.save_for_backward(codes, scales)
        ctx.K = K
        return _product("gdn_mxfp4_linear", x, Weight(codes, scales, K), False)

    @staticmethod
    def backward(ctx, dy):
        codes, scales = ctx.saved_tensors
        dx = _product("gdn_mxfp4_linear_bwd", dy, Weight(codes, scales, ctx.K), True)
        return (*L.once((dy,), dx), None, None, None)


def linear(x: Array, q: Weight) -> Array:
    """``x`` [..., K] times the weight's transpose: [..., N] of x's type, rounded once from 32-bit sums that the weight's values
    and all bits of ``x`` enter.  Differentiable in ``x``; the weight is frozen.  At most 64 rows read the 4-bit weight itself
    (no workspace); more need a bf16 copy of it for the time of the call, as does the gradient, 2^26 elements at a time."""
    _check(q)
    if x.dim() < 1 or x.shape[-1] != q.columns:
        raise ValueError(f"x must be [..., {q.columns}]; got {tuple(x.shape)}")
    if x.dtype not in L.DTYPE_CODE:
        raise ValueError(f"unsupported dtype {x.dtype}; use float32, bfloat16 or float16")
    L.refuse_tangents("linear", x)
    _on_gpu(x, "linear")
    if q.codes.device != x.device:
        raise ValueError("all inputs must be on the same device")
    if q.codes.shape[0] == 0:
        raise ValueError("the weight must have rows")
    lead = x.shape[:-1]
    rows = x if x.dim() == 2 else x.reshape(-1, q.columns)
    if torch.is_grad_enabled() and x.requires_grad:
        y = _Linear.apply(rows, *q)
    else:
        y = _product("gdn_mxfp4_linear", rows, q, False)
    return y if x.dim() == 2 else y.view(*lead, y.shape[1])


class MXFP4Linear(torch.nn.Module):
    """A frozen bias-free linear layer with its weight in MXFP4."""

    def __init__(self, q: Weight):
        super().__init__()
        _check(q)
        self.out_features, self.in_features = q.shape
        self.register_buffer("codes", q.codes)
        self.register_buffer("scales", q.scales)

    @classmethod
    def of(cls, m: torch.nn.Linear) -> "MXFP4Linear":
        if m.bias is not None:
            raise ValueError("layers with a bias are not supported")
        return cls(quantize(m.weight))

    def forward(self, x: Array) -> Array:
        return linear(x, Weight(self.codes, self.scales, self.in_features))
