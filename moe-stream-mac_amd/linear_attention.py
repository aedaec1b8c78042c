"""Linear attention with a log decay for each head: whole sequences (a prompt, a training step) and single tokens.

    S_t = e^{g_t} S_{t-1} + v_t k_t^T,    y_t = scale S_t q_t

The recurrence of the GDN layers without their delta rule, in HIP kernels: a chunked form on the matrix cores with its
backward pass, and a recurrent step for decoding.  Tensors must live on a ROCm device; there is no CPU path.
"""

from __future__ import annotations

import contextlib
import ctypes
from typing import Optional

import torch

import gdn_lib as L

Array = torch.Tensor


def _check(q: Array, k: Array, v: Array, g: Array, state: Optional[Array], lead: int) -> None:
    """Shapes of q, k [*lead, Hk, Dk], v [*lead, Hv, Dv], g [*lead, Hv] or [Hv], state [B, Hv, Dv, Dk]."""
    names = "[B, T" if lead == 2 else "[B"
    if q.dim() != lead + 2 or k.shape != q.shape:
        raise ValueError(f"q and k must both be {names}, Hk, Dk]; got {tuple(q.shape)}, {tuple(k.shape)}")
    if v.dim() != lead + 2 or v.shape[:lead] != q.shape[:lead]:
        raise ValueError(f"v must be {names}, Hv, Dv]; got {tuple(v.shape)} for q {tuple(q.shape)}")
    B, (Hk, Dk), (Hv, Dv) = q.shape[0], q.shape[lead:], v.shape[lead:]
    if min(Hk, Dk, Hv, Dv) < 1 or Hv % Hk:
        raise ValueError(f"the key heads must divide the value heads; got {Hk} and {Hv}")
    if tuple(g.shape) not in ((Hv,), (*q.shape[:lead], Hv)):
        raise ValueError(f"g must be [Hv] or {names}, Hv] = {(*q.shape[:lead], Hv)}; got {tuple(g.shape)}")
    if q.dtype != k.dtype or q.dtype != v.dtype or q.dtype not in L.DTYPE_CODE:
        raise ValueError(f"q, k and v must share one of float32, bfloat16, float16; got {q.dtype}, {k.dtype}, {v.dtype}")
    if g.dtype not in L.DTYPE_CODE:
        raise ValueError(f"unsupported dtype {g.dtype} of g; use float32, bfloat16 or float16")
    if state is not None and tuple(state.shape) != (B, Hv, Dv, Dk):
        raise ValueError(f"state must be [B, Hv, Dv, Dk] = {(B, Hv, Dv, Dk)}; got {tuple(state.shape)}")
    if q.device.type != "cuda":
        raise RuntimeError("linear attention runs on a ROCm GPU only; got tensors on " + str(q.device))
    if any(t is not None and t.device != q.device for t in (k, v, g, state)):
        raise ValueError("all inputs must be on the same device")


def _rows(t: Array) -> Array:
    """t with channels side by side and tokens less than 2^22 elements apart, what the kernels take."""
    return t if (t.stride(-1) == 1 or t.shape[-1] == 1) and t.stride(1) < 1 << 22 else t.contiguous()


def _strides(q: Array, k: Array, v: Array, g: Array):
    gs = (0, 0, g.stride(0)) if g.dim() == 1 else g.stride()
    return (ctypes.c_int64 * 12)(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *gs)


def _forward(q, k, v, g, state, scale):
    """y, the final state and what the backward needs of the states between."""
    (B, T, Hk, Dk), (Hv, Dv), dev = q.shape, v.shape[2:], q.device
    y = torch.empty((B, T, Hv, Dv), dtype=q.dtype, device=dev)
    last = torch.empty((B, Hv, Dv, Dk), dtype=torch.float32, device=dev)
    lib = L.load()
    n = lib.gdn_linatt_saved_bytes(B, T, Hk, Hv, Dk, Dv)
    saved = torch.empty((n,), dtype=torch.uint8, device=dev)
    with L.on_device(dev):
        L.check(lib.gdn_linatt_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), L.ptr(state), y.data_ptr(),
                                   last.data_ptr(), saved.data_ptr(), n, _strides(q, k, v, g), B, T, Hk, Hv, Dk, Dv, scale,
                                   L.DTYPE_CODE[q.dtype], L.DTYPE_CODE[g.dtype], L.stream_handle(dev)))
    return y, last, saved


class _LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, state, scale):
        ctx.set_materialize_grads(False)
        y, last, saved = _forward(q, k, v, g, state, scale)
        ctx.save_for_backward(q, k, v, g, state, last, saved)
        ctx.scale = scale
        return y, last

    @staticmethod
    def backward(ctx, dy, dlast):
        q, k, v, g, state, last, saved = ctx.saved_tensors
        (B, T, Hk, Dk), (Hv, Dv), dev = q.shape, v.shape[2:], q.device
        if dy is None and dlast is None:
            return (None,) * 6
        dy = torch.zeros((B, T, Hv, Dv), dtype=q.dtype, device=dev) if dy is None else dy.contiguous()
        dlast = None if dlast is None else dlast.contiguous()
        dq, dk = (torch.empty((B, T, Hk, Dk), dtype=q.dtype, device=dev) for _ in range(2))
        dv = torch.empty((B, T, Hv, Dv), dtype=q.dtype, device=dev)
        dg = torch.empty(g.shape, dtype=g.dtype, device=dev)
        dstate = torch.empty_like(state) if ctx.needs_input_grad[4] else None
        lib = L.load()
        n = lib.gdn_linatt_bwd_workspace_bytes(B, T, Hk, Hv, Dk, Dv, L.DTYPE_CODE[q.dtype])
        ws = torch.empty((n,), dtype=torch.uint8, device=dev)
        with L.on_device(dev):
            L.check(lib.gdn_linatt_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), L.ptr(state), last.data_ptr(),
                                       saved.data_ptr(), saved.numel(), dy.data_ptr(), L.ptr(dlast),
                                       dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dg.data_ptr(), L.ptr(dstate),
                                       ws.data_ptr(), n, _strides(q, k, v, g), B, T, Hk, Hv, Dk, Dv, ctx.scale,
                                       int(g.dim() == 1), L.DTYPE_CODE[q.dtype], L.DTYPE_CODE[g.dtype],
                                       L.stream_handle(dev)))
        return (*L.once((q, k, v, g, state, dy, dlast), dq, dk, dv, dg, dstate), None)


def linear_attention(q: Array, k: Array, v: Array, g: Array, state: Optional[Array] = None, *,
                     scale: Optional[float] = None) -> tuple[Array, Array]:
    """(y [B, T, Hv, Dv] in q's type, final state [B, Hv, Dv, Dk] in float32) from q, k [B, T, Hk, Dk], v [B, T, Hv, Dv]
    and the log decays ``g`` [B, T, Hv], or [Hv] for one of each head; value head h reads key head h / (Hv / Hk).

    ``state`` is the state before the first token (None: zeros), ``scale`` defaults to Dk^-1/2.  A log decay of -inf keeps
    nothing of the state.  q, k, v and g may be strided views; heads have at most 256 channels.  Differentiable in q, k, v, g
    and state (once: no second derivatives); gradients have their inputs' types.

    An infinite or NaN input of one token does not reach the outputs before it, nor gradients that it has no part in; what it
    has a part in may be NaN where the formula gives an infinity.  Decays' gradients that lie between two such tokens less than
    512 apart may be NaN as well, and one log decay for a head has the sum of all its tokens' gradients."""
    _check(q, k, v, g, state, 2)
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    if q.shape[0] == 0 or q.shape[1] == 0:  # no token: the state passes through
        B, (Hv, Dv) = q.shape[0], v.shape[2:]
        last = q.new_zeros((B, Hv, Dv, q.shape[-1]), dtype=torch.float32) if state is None else state.float().clone()
        return v.new_empty((*q.shape[:2], Hv, Dv)), last
    q, k, v = _rows(q), _rows(k), _rows(v)
    state = None if state is None else state.float().contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, g, state)):
        return _LinearAttention.apply(q, k, v, g, state, scale)
    return _forward(q, k, v, g, state, scale)[:2]


class _NoGradient(torch.autograd.Function):
    """A result of a step as autograd sees it: it depends on the step's inputs, and a gradient through it is refused."""

    @staticmethod
    def forward(ctx, result, *inputs):
        ctx.mark_dirty(result)
        return result

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError("linear_attention_step is not differentiable; use linear_attention")


def linear_attention_step(q: Array, k: Array, v: Array, g: Array, state: Array, *,
                          scale: Optional[float] = None) -> Array:
    """One token of B sequences: q, k [B, Hk, Dk], v [B, Hv, Dv], g [B, Hv] or [Hv].  Updates ``state`` [B, Hv, Dv, Dk]
    (contiguous float32) in place and returns y [B, Hv, Dv].  Not differentiable: with gradients enabled, a backward pass
    that reaches a step whose inputs require them raises."""
    _check(q, k, v, g, state, 1)
    if state.dtype != torch.float32 or not state.is_contiguous():
        raise ValueError("state must be contiguous float32: it is updated in place")
    (B, Hk, Dk), (Hv, Dv), dev = q.shape, v.shape[1:], q.device
    inputs = (q, k, v, g, state) if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, g, state)) else None
    if inputs:
        # torch itself refuses leaves and views made without gradients, whose earlier uses the change of version guards
        with contextlib.suppress(RuntimeError):
            _NoGradient.apply(state, q, k, v, g)
    # the copies stay referenced until the launch is enqueued
    q, k, v, g = q.detach().contiguous(), k.detach().contiguous(), v.detach().contiguous(), g.detach()
    y = torch.empty((B, Hv, Dv), dtype=q.dtype, device=dev)
    gs = (0, g.stride(0)) if g.dim() == 1 else g.stride()
    with L.on_device(dev):
        L.check(L.load().gdn_linatt_step(q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), state.data_ptr(),
                                         y.data_ptr(), *gs, B, Hk, Hv, Dk, Dv,
                                         Dk ** -0.5 if scale is None else float(scale), L.DTYPE_CODE[q.dtype],
                                         L.DTYPE_CODE[g.dtype], L.stream_handle(dev)))
    L.written((state,))
    return _NoGradient.apply(y, *inputs) if inputs else y
