"""ctypes binding to ``libgdn_mi355x.so`` (C ABI declared in ``include/gdn_mi355x.h``).

torch is imported before the library is opened so that the library binds to the HIP runtime torch already
loaded (both carry the soname ``libamdhip64.so.7``); device pointers and streams are then shared.
There is no fallback: a missing library is an error.
"""

from __future__ import annotations

import contextlib
import ctypes
import os
import re
from pathlib import Path

import torch  # noqa: F401  (must precede loading the HIP library)
import torch.autograd.forward_ad as fwAD

LIB_PATH = Path(__file__).resolve().parent / "libgdn_mi355x.so"
HEADER = Path(__file__).resolve().parent.parent / "include" / "gdn_mi355x.h"

GDN_OK, GDN_ERR_INVALID, GDN_ERR_UNSUPPORTED, GDN_ERR_WORKSPACE, GDN_ERR_LAUNCH = 0, -1, -2, -3, -4
F32, BF16, F16 = 0, 1, 2
GATE_DECAY, GATE_DECAY_VEC, GATE_LOG, GATE_LOG_VEC = 0, 1, 2, 3
FORM_AUTO, FORM_RECURRENT, FORM_CHUNK = 0, 1, 2
FORMS = {"auto": FORM_AUTO, "recurrent": FORM_RECURRENT, "chunk": FORM_CHUNK}

DTYPE_CODE = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}

_vp = ctypes.c_void_p
_i = ctypes.c_int
_i64 = ctypes.c_int64
_f = ctypes.c_float
_d = ctypes.c_double
_sz = ctypes.c_size_t
_SIGS = {
    "gdn_gates_fwd": ([_vp] * 6 + [_i64, _i, _i, _i, _i, _vp], _i),
    "gdn_gates_bwd_workspace_bytes": ([_i64, _i], _sz),
    "gdn_gates_bwd": ([_vp] * 12 + [_sz, _i64, _i, _i, _i, _i, _i, _vp], _i),
    "gdn_l2norm_fwd": ([_vp, _vp, _i64, _i, _f, _f, _i, _vp], _i),
    "gdn_l2norm_bwd": ([_vp, _vp, _vp, _i64, _i, _f, _f, _i, _i, _vp], _i),
    "gdn_conv_silu_fwd": ([_vp] * 5 + [_i] * 5 + [_vp], _i),
    "gdn_conv_silu_bwd_workspace_bytes": ([_i] * 4, _sz),
    "gdn_conv_silu_bwd": ([_vp] * 7 + [_sz] + [_i] * 6 + [_vp], _i),
    "gdn_conv_qkv_fwd": ([_vp] * 7 + [_i] * 7 + [_f, _f, _i, _vp], _i),
    "gdn_conv_qkv_bwd": ([_vp] * 9 + [_sz] + [_i] * 7 + [_f, _f, _i, _i, _vp], _i),
    "gdn_gated_rmsnorm_fwd": ([_vp] * 4 + [_i64, _i, _f, _i, _i, _vp], _i),
    "gdn_gated_rmsnorm_bwd_workspace_bytes": ([_i64, _i], _sz),
    "gdn_gated_rmsnorm_bwd": ([_vp] * 8 + [_sz, _i64, _i, _f, _i, _i, _i, _vp], _i),
    "gdn_small_linears": ([_vp] * 4 + [_i] * 4 + [_vp], _i),
    "gdn_block_decode": ([_vp] * 13 + [_i] * 11 + [_f] * 3 + [_vp], _i),
    "gdn_rotary": ([_vp] * 6 + [_i64] * 8 + [_i] * 9 + [_f, _i, _vp], _i),
    "gdn_logprobs_workspace_bytes": ([_i64, _i64, _i], _sz),
    "gdn_logprobs_fwd": ([_vp] * 8 + [_sz] + [_i64] * 6 + [_i, _i, _vp], _i),
    "gdn_logprobs_bwd": ([_vp] * 7 + [_i64] * 6 + [_i, _vp], _i),
    "gdn_clip_grad_norm_workspace_bytes": ([_vp, _i], _sz),
    "gdn_clip_grad_norm": ([_vp] * 4 + [_i, _i, _d, _d, _vp, _vp, _sz, _vp], _i),
    "gdn_linatt_saved_bytes": ([_i] * 6, _sz),
    "gdn_linatt_bwd_workspace_bytes": ([_i] * 7, _sz),
    "gdn_linatt_fwd": ([_vp] * 8 + [_sz, _vp] + [_i] * 6 + [_f, _i, _i, _vp], _i),
    "gdn_linatt_bwd": ([_vp] * 7 + [_sz] + [_vp] * 8 + [_sz, _vp] + [_i] * 6 + [_f, _i, _i, _i, _vp], _i),
    "gdn_linatt_step": ([_vp] * 6 + [_i64, _i64] + [_i] * 5 + [_f, _i, _i, _vp], _i),
    "gdn_linear_loss_workspace_bytes": ([_i64] * 3 + [_i] * 4, _sz),
    "gdn_linear_loss_fwd": ([_vp] * 8 + [_sz] + [_i64] * 6 + [_i, _i, _vp], _i),
    "gdn_linear_loss_bwd": ([_vp] * 5 + [_i64] + [_vp] * 4 + [_sz] + [_i64] * 6 + [_i, _vp], _i),
    "gdn_embedding_fwd": ([_vp] * 3 + [_i64] * 4 + [_d, _i, _vp], _i),
    "gdn_embedding_bwd_workspace_bytes": ([_i64] * 3, _sz),
    "gdn_embedding_bwd": ([_vp] * 4 + [_sz] + [_i64] * 5 + [_d, _i, _vp], _i),
    "gdn_mxfp4_quantize": ([_vp] * 3 + [_i64] * 3 + [_i, _vp], _i),
    "gdn_mxfp4_dequantize": ([_vp] * 3 + [_i64] * 2 + [_i, _vp], _i),
    "gdn_mxfp4_linear_workspace_bytes": ([_i64] * 3 + [_i] * 3, _sz),
    "gdn_mxfp4_linear": ([_vp] * 5 + [_sz] + [_i64] * 4 + [_i, _vp], _i),
    "gdn_mxfp4_linear_bwd": ([_vp] * 5 + [_sz] + [_i64] * 4 + [_i, _vp], _i),
    "gdn_version": ([], _i),
    "gdn_last_error": ([], ctypes.c_char_p),
    "gdn_num_snapshots": ([_i, _i], ctypes.c_int64),
    "gdn_select_form": ([_i] * 7, _i),
    "gdn_saved_bytes": ([_i] * 11, ctypes.c_size_t),
    "gdn_fwd_workspace_bytes": ([_i] * 12, ctypes.c_size_t),
    "gdn_fwd": ([_vp] * 10 + [_sz, _vp, _sz] + [_i] * 11 + [_vp], _i),
    "gdn_bwd_workspace_bytes": ([_i] * 11, ctypes.c_size_t),
    "gdn_decode_step": ([_vp] * 8 + [_i] * 8 + [_vp], _i),
    "gdn_fwd_noalloc": ([_vp] * 9 + [_i] * 10 + [_vp], _i),
    "gdn_bwd": ([_vp] * 8 + [ctypes.c_size_t] + [_vp] * 9 + [ctypes.c_size_t] + [_i] * 12 + [_vp], _i),
    "gdn_profile_enable": ([_i], _i),
    "gdn_profile_collect": ([_i, ctypes.c_char_p, _i, ctypes.POINTER(ctypes.c_double),
                             ctypes.POINTER(_i)], _i),
}

_lib = None


class GDNError(RuntimeError):
    """A non-zero status from the C ABI."""

    def __init__(self, status: int, message: str):
        super().__init__(message)
        self.status = status


def load() -> ctypes.CDLL:
    """Open the library once; raises if it was never built."""
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise RuntimeError(
                f"{LIB_PATH} is missing: build the HIP engine first "
                "(python moe-stream-mac_amd/build.py or __graft_entry__.build())")
        lib = ctypes.CDLL(os.fspath(LIB_PATH), mode=ctypes.RTLD_GLOBAL)
        for name, (args, res) in _SIGS.items():
            fn = getattr(lib, name)
            fn.argtypes = args
            fn.restype = res
        _lib = lib
    return _lib


def header_functions() -> list[str]:
    """Function names declared by include/gdn_mi355x.h."""
    text = HEADER.read_text()
    return sorted(set(re.findall(r"^\s*(?:const\s+)?[a-z_0-9]+\s*\*?\s*(gdn_[a-z_0-9]+)\s*\(", text, re.M)))


def check(status: int) -> None:
    if status != GDN_OK:
        msg = load().gdn_last_error().decode(errors="replace")
        if status in (GDN_ERR_INVALID,):
            raise ValueError(msg)
        raise GDNError(status, msg)


def ptr(t) -> int | None:
    return None if t is None else t.data_ptr()


MOST_PITCH = 1 << 23  # bytes between the rows of an operand that a matrix product reads as it lies


def row_stride(t) -> int:
    """Elements from row to row of a matrix with contiguous channels."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def rows_lie_well(*rows) -> bool:
    """Whether matrix products may read these matrices as they lie, which the workspace queries call aligned."""
    return all(t.data_ptr() % 16 == 0 and row_stride(t) * t.element_size() % 16 == 0
               and row_stride(t) * t.element_size() <= MOST_PITCH for t in rows)


def written(tensors) -> None:
    """Tensors that a kernel changed in place: autograd refuses to go back through what had saved their old values."""
    torch.autograd.graph.increment_version(tensors)


def refuse_tangents(what: str, *tensors) -> None:
    """Raises where a tensor carries a forward-mode tangent: a kernel sees the primal alone, and its result would be a constant."""
    if fwAD._current_level >= 0 and any(t is not None and fwAD.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{what} has no forward-mode derivative")


class _Once(torch.autograd.Function):
    @staticmethod
    def forward(ctx, n, *inputs_and_grads):
        return inputs_and_grads[n:]

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("gradients of this operator cannot be differentiated twice")


def once(inputs, *grads):
    """A backward pass's results: with create_graph, ones that raise when they are differentiated in what they depend on,
    its ``inputs``, instead of constants.  Forward-mode tangents of the inputs are refused."""
    refuse_tangents("a gradient of this operator", *inputs)
    return _Once.apply(len(inputs), *inputs, *grads) if torch.is_grad_enabled() else grads


def profile_enable(on: bool) -> None:
    load().gdn_profile_enable(1 if on else 0)


def profile_collect() -> dict[str, tuple[float, int]]:
    """{kernel: (total_ms, launches)} recorded since the last collect (waits for the events)."""
    n_max, name_len = 32, 64
    names = ctypes.create_string_buffer(n_max * name_len)
    ms = (ctypes.c_double * n_max)()
    counts = (ctypes.c_int * n_max)()
    n = load().gdn_profile_collect(n_max, names, name_len, ms, counts)
    if n < 0:
        check(n)
    out = {}
    for i in range(n):
        raw = names.raw[i * name_len:(i + 1) * name_len]
        out[raw.split(b"\0", 1)[0].decode()] = (ms[i], counts[i])
    return out


def on_device(dev: torch.device):
    """A context in which launches go to ``dev``: nothing where it is the current device already."""
    return contextlib.nullcontext() if dev.index in (None, torch.cuda.current_device()) else torch.cuda.device(dev)


def stream_handle(device: torch.device) -> int:
    if device.index is None:
        return torch.cuda.current_stream(device).cuda_stream
    # without a Stream object around it (3 us each)
    return torch._C._cuda_getCurrentRawStream(device.index)
