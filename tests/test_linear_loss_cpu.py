"""Refusals and host logic of the cross entropy without logits (no kernel launches)."""

import ctypes

import pytest
import torch

import gdn_lib as L


def test_abi_refusals():
    lib = L.load()
    fake = ctypes.c_void_p(4096)  # never dereferenced: every call fails its checks first

    def fwd(N=4, H=64, V=100, xs=64, ws=64, red=0, dt=1, p=fake, total=fake, room=1 << 40):
        return lib.gdn_linear_loss_fwd(p, p, p, p, p, total, total, p, room, N, H, V, xs, ws, -100, red, dt, None)

    for kw in (dict(N=-1), dict(H=0), dict(V=0), dict(dt=3), dict(red=3), dict(red=1, total=None), dict(p=None), dict(xs=63),
               dict(ws=10)):
        assert fwd(**kw) == L.GDN_ERR_INVALID, kw
    for kw in (dict(N=(1 << 20) + 1), dict(V=(1 << 24) + 1), dict(H=(1 << 17) + 1, xs=1 << 18, ws=1 << 18)):
        assert fwd(**kw) == L.GDN_ERR_UNSUPPORTED, kw
    need = lib.gdn_linear_loss_workspace_bytes(4, 64, 100, 1, 1, 0, 0)
    assert need > 0 and fwd(room=need - 1) == L.GDN_ERR_WORKSPACE and b"workspace" in lib.gdn_last_error()
    assert fwd(N=0, p=None) == 0
    assert lib.gdn_linear_loss_workspace_bytes(0, 64, 100, 1, 1, 0, 0) == 0

    def bwd(N=4, dt=1, p=fake, dx=fake, dw=fake, stride=1, room=1 << 40):
        return lib.gdn_linear_loss_bwd(p, p, p, p, p, stride, None, dx, dw, p, room, N, 64, 100, 64, 64, -100, dt, None)

    assert bwd(dx=None, dw=None) == 0
    for kw in (dict(N=0), dict(p=None), dict(stride=2), dict(dt=9), dict(N=-3)):
        assert bwd(**kw) == L.GDN_ERR_INVALID, kw
    for dx, dw in ((fake, None), (None, fake), (fake, fake)):
        need = lib.gdn_linear_loss_workspace_bytes(4, 64, 100, 1, 1, dx is not None, dw is not None)
        assert bwd(dx=dx, dw=dw, room=need - 1) == L.GDN_ERR_WORKSPACE


def test_workspace_stays_bounded():
    """Forward 2^26 statistics or 256 tokens', the tokens that count with their places, and room for copies of what is not
    aligned; backward 2^26 differences, in 16 bits for each gradient, or 256 words', the operands of their products and fp32 sums
    of dx in parts."""
    f, H, MB = L.load().gdn_linear_loss_workspace_bytes, 2048, 1 << 20
    for N, V in ((8192, 131072), (1 << 20, 131072), (1 << 20, 1000), (100, 1 << 24)):
        stats = 8 * max(1 << 26, 256 * (V // 64 + 512))
        chosen = N * (16 + 2 * H) if N >= 2048 else 0
        assert f(N, H, V, 1, 1, 0, 0) <= stats + 4 * N + chosen + MB, (N, V)
        assert f(N, H, V, 1, 0, 0, 0) <= stats + 20 * N + 2 * H * (N + min(V, (1 << 26) // N + 512)) + MB
        words = min(V, max(256, (1 << 26) // N) + 512)
        sums = 4 * N * H * max(1, min(16, 256 // (8 * (N // 256 + 1)) + 1))
        back = 4 * words * (N + 64) + 2 * H * (words + 64) + 2 * H * (N + 64) + 4 * N + sums + 8 * 4 * words * H + chosen + MB
        assert f(N, H, V, 1, 1, 1, 1) <= back, (N, V)
    # a long batch: an eighth of the logits in 16 bits
    assert f(65536, H, 131072, 1, 1, 1, 0) < 65536 * 131072 * 2 / 8


def test_wrapper_refuses():
    from linear_loss import linear_cross_entropy
    x, w, t = torch.zeros(2, 3, 8), torch.zeros(10, 8), torch.zeros(2, 3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        linear_cross_entropy(x, w, t)
    for bad in (lambda: linear_cross_entropy(x[..., :7], w, t), lambda: linear_cross_entropy(x, w[0], t),
                lambda: linear_cross_entropy(x, w, t[:1]), lambda: linear_cross_entropy(x.half(), w, t),
                lambda: linear_cross_entropy(x.double(), w.double(), t), lambda: linear_cross_entropy(x, w, t.float()),
                lambda: linear_cross_entropy(x, w[:0], t), lambda: linear_cross_entropy(x, w, t, reduction="max")):
        with pytest.raises(ValueError):
            bad()
