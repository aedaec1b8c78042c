"""The global norm of a model's gradients, and the gradients scaled by it: a few launches for any number of tensors, no
synchronisation with the host.  Tensors must live on a ROCm device; there is no CPU path.
"""

from __future__ import annotations

import math
from array import array
from operator import attrgetter
from typing import Iterable, Optional

import torch

import gdn_lib as L

Array = torch.Tensor

# a model has hundreds of tensors: attributes are taken by maps, without a line of Python for each
_layout, _dtype, _shape = attrgetter("layout"), attrgetter("dtype"), attrgetter("shape")
_index, _numel, _ptr, _contiguous = Array.get_device, Array.numel, Array.data_ptr, Array.is_contiguous


def _dense(t: Array) -> bool:
    """Whether the tensor fills a block of memory in some order of its axes (a transposed weight does)."""
    if t.is_contiguous():
        return True
    want = 1
    for n, s in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n != 1), key=lambda p: p[1]):
        if s != want:
            return False
        want *= n
    return True


def _check(tensors, norm_type) -> None:
    if norm_type not in (2.0, math.inf):
        raise ValueError(f"norm_type must be 2 or inf; got {norm_type}")
    if set(map(_layout, tensors)) != {torch.strided} or not set(map(_dtype, tensors)) <= L.DTYPE_CODE.keys():
        t = next(t for t in tensors if t.layout != torch.strided or t.dtype not in L.DTYPE_CODE)
        raise ValueError(f"unsupported tensor ({t.dtype}, {t.layout}); use dense float32, bfloat16 or float16")
    if len(set(map(_index, tensors))) > 1:
        raise ValueError("all tensors must be on the same device")
    if tensors[0].device.type != "cuda":
        raise RuntimeError("grad_clip runs on a ROCm GPU only; got tensors on " + str(tensors[0].device))


def _same_dtypes(a, b) -> bool:
    one = set(map(_dtype, a))
    return set(map(_dtype, b)) == one and (len(one) == 1 or list(map(_dtype, a)) == list(map(_dtype, b)))


def _call(tensors, outs, max_norm, norm_type, eps) -> Array:
    dev, n = tensors[0].device, len(tensors)
    dtypes = set(map(_dtype, tensors))
    if len(dtypes) == 1:
        codes = array("i", [L.DTYPE_CODE[dtypes.pop()]]) * n
    else:
        codes = array("i", map(L.DTYPE_CODE.__getitem__, map(_dtype, tensors)))
    numel, x = array("q", map(_numel, tensors)), array("Q", map(_ptr, tensors))
    y = None if outs is None else x if outs is tensors else array("Q", map(_ptr, outs))
    at = lambda a: a.buffer_info()[0]  # noqa: E731  (the arrays live until the call is over)
    lib = L.load()
    norm = torch.empty((), dtype=torch.float32, device=dev)
    nws = lib.gdn_clip_grad_norm_workspace_bytes(at(numel), n)
    ws = torch.empty((nws,), dtype=torch.uint8, device=dev)
    with L.on_device(dev):
        L.check(lib.gdn_clip_grad_norm(at(x), None if y is None else at(y), at(numel), at(codes), n,
                                       int(norm_type == math.inf), float(max_norm), float(eps), norm.data_ptr(),
                                       ws.data_ptr(), nws, L.stream_handle(dev)))
    return norm


def grad_norm(tensors: Iterable[Array], norm_type: float = 2.0) -> Array:
    """The norm over all elements of all tensors: 2 (squares summed in 64 bits) or inf; a float32 scalar on the device."""
    ts = list(tensors)
    if not ts:
        return torch.zeros(())
    _check(ts, norm_type)
    return _call([t if _dense(t) else t.contiguous() for t in ts], None, 0.0, float(norm_type), 0.0)


def clip_grad_norm(grads: Iterable[Array], max_norm: float, norm_type: float = 2.0, *,
                   out: Optional[Iterable[Array]] = None, eps: float = 1e-6) -> Array:
    """Multiplies every tensor by min(1, max_norm / (norm + eps)) in place, or into the tensors of ``out`` (same shapes
    and types), and returns the norm over all of them before that, as a float32 scalar on the device.  ``norm_type`` is 2
    or inf.  A NaN in any tensor makes the norm and every result NaN; an infinite norm scales by 0.  Tensors may differ
    in type and have any strides; none may share memory with another that is written.  Not differentiable."""
    gs = list(grads)
    if not max_norm >= 0:
        raise ValueError(f"max_norm must be >= 0; got {max_norm}")
    if not eps >= 0:
        raise ValueError(f"eps must be >= 0; got {eps}")
    if not gs:
        return torch.zeros(())
    _check(gs, norm_type)
    os_ = gs if out is None else list(out)
    if out is not None and (list(map(_shape, os_)) != list(map(_shape, gs)) or
                            not _same_dtypes(gs, os_) or
                            set(map(_index, os_)) != {gs[0].get_device()} or set(map(_layout, os_)) != {torch.strided}):
        raise ValueError("out must hold one tensor of the same shape, type and device for each gradient")
    if all(map(_contiguous, gs)) and (os_ is gs or all(map(_contiguous, os_))):
        norm = _call(gs, os_, max_norm, float(norm_type), eps)
        L.written(os_)
        return norm
    # memory order does not matter to the kernels where input and output share it; others go through a copy
    src, dst, back = [], [], []
    for g, o in zip(gs, os_):
        g, o = g.detach(), o.detach()
        if (g.is_contiguous() and o.is_contiguous()) or (_dense(g) and g.stride() == o.stride()):
            src.append(g)
            dst.append(o)
        else:
            src.append(g.contiguous())
            dst.append(torch.empty_like(src[-1]))
            back.append((o, dst[-1]))
    norm = _call(src, dst, max_norm, float(norm_type), eps)
    for o, tmp in back:
        o.copy_(tmp)
    L.written(os_)
    return norm
