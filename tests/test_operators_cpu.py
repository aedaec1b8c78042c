"""Refusals and host logic of the language-model operators (no kernel launches)."""

import ctypes
import math

import pytest
import torch

import gdn_lib as L


def test_rotary_abi_refusals():
    lib = L.load()
    fake = ctypes.c_void_p(256)  # never dereferenced: every call fails its checks first

    def call(B=1, T=4, Hq=2, Hk=1, D=64, R=64, dt=0, p=fake):
        return lib.gdn_rotary(p, p, p, p, p, p, *[1] * 8, B, T, Hq, Hk, D, R, 0, 0, 1, 1.0, dt, None)

    assert call(B=-1) == L.GDN_ERR_INVALID and call(D=0) == L.GDN_ERR_INVALID
    assert call(R=0) == L.GDN_ERR_INVALID and call(R=3) == L.GDN_ERR_INVALID and call(R=66) == L.GDN_ERR_INVALID
    assert call(D=4096, R=2048) == L.GDN_ERR_UNSUPPORTED
    assert call(dt=3) == L.GDN_ERR_INVALID
    assert call(p=None) == L.GDN_ERR_INVALID and b"null" in lib.gdn_last_error()
    assert call(T=0, p=None) == 0 and call(Hq=0, Hk=0, p=None) == 0


def test_logprobs_abi_refusals():
    lib = L.load()
    fake = ctypes.c_void_p(256)

    def fwd(outer=1, inner=4, V=100, top=0, dt=0, ws=1 << 40, p=fake):
        return lib.gdn_logprobs_fwd(p, p, p, p, p, p, p, p, ws, outer, inner, V, 0, V, -100, top, dt, None)

    assert fwd(V=0) == L.GDN_ERR_INVALID and fwd(outer=-1) == L.GDN_ERR_INVALID and fwd(dt=7) == L.GDN_ERR_INVALID
    assert fwd(top=101) == L.GDN_ERR_INVALID and fwd(top=-1) == L.GDN_ERR_INVALID
    assert fwd(top=65) == L.GDN_ERR_UNSUPPORTED
    assert fwd(V=8192 * 128 + 1, top=64) == L.GDN_ERR_UNSUPPORTED
    assert fwd(outer=1 << 20, inner=32) == L.GDN_ERR_UNSUPPORTED
    assert fwd(ws=lib.gdn_logprobs_workspace_bytes(4, 100, 0) - 1) == L.GDN_ERR_WORKSPACE
    assert fwd(p=None) == L.GDN_ERR_INVALID
    assert fwd(outer=0, p=None) == 0
    bwd = lambda p, s, e: lib.gdn_logprobs_bwd(p, p, s, e, p, p, p, 1, 4, 100, 0, 100, -100, 0, None)  # noqa: E731
    assert bwd(fake, None, fake) == L.GDN_ERR_INVALID and bwd(fake, fake, None) == L.GDN_ERR_INVALID


def test_clip_abi_refusals():
    lib = L.load()
    fake = 4096

    def call(xs, ys, sizes, dts, max_norm=1.0, ws=1 << 40, norm=fake, inf=0):
        n = len(sizes)
        return lib.gdn_clip_grad_norm((ctypes.c_void_p * n)(*xs), None if ys is None else (ctypes.c_void_p * n)(*ys),
                                      (ctypes.c_int64 * n)(*sizes), (ctypes.c_int * n)(*dts), n, inf, max_norm, 1e-6,
                                      norm, fake, ws, None)

    assert call([fake], None, [-1], [0]) == L.GDN_ERR_INVALID
    assert call([fake], None, [5], [9]) == L.GDN_ERR_INVALID
    assert call([None], None, [5], [0]) == L.GDN_ERR_INVALID
    assert call([fake], [None], [5], [0]) == L.GDN_ERR_INVALID
    assert call([fake], [fake], [5], [0], max_norm=-1.0) == L.GDN_ERR_INVALID
    assert call([fake], [fake], [5], [0], max_norm=math.nan) == L.GDN_ERR_INVALID
    assert call([fake], None, [5], [0], norm=None) == L.GDN_ERR_INVALID
    assert call([fake], None, [5], [0], ws=8) == L.GDN_ERR_WORKSPACE
    # two outputs, an output and another's input, an output across its own input
    assert call([fake, fake + 16], [fake, fake + 16], [5, 5], [0, 0]) == L.GDN_ERR_INVALID
    assert b"share memory" in lib.gdn_last_error()
    assert call([4096, 8192], [8192, 1 << 20], [5, 5], [0, 0]) == L.GDN_ERR_INVALID
    assert call([4096], [4100], [5], [0]) == L.GDN_ERR_INVALID
    # neighbours that only touch pass this check (and fail the workspace's)
    assert call([4096, 4106], [4096, 4106], [5, 5], [1, 1], ws=0) == L.GDN_ERR_WORKSPACE


def test_wrappers_refuse():
    from grad_clip import clip_grad_norm, grad_norm
    from rotary import rotary, rotary_frequencies
    from token_logprobs import token_logprobs
    q, pos = torch.zeros(1, 3, 2, 8), torch.arange(3)
    inv, _ = rotary_frequencies(8)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        rotary(q, q, pos, inv)
    for bad in (lambda: rotary(q, q[:, :2], pos, inv), lambda: rotary(q, q, pos[:2], inv),
                lambda: rotary(q, q, pos.float(), inv), lambda: rotary(q, q.half(), pos, inv),
                lambda: rotary(q, q, pos, torch.ones(5)), lambda: rotary(q.int(), q.int(), pos, inv)):
        with pytest.raises(ValueError):
            bad()
    z, y = torch.zeros(2, 10), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        token_logprobs(z, y)
    for bad in (lambda: token_logprobs(z, y[:1]), lambda: token_logprobs(z, y, top=11),
                lambda: token_logprobs(z.double(), y), lambda: token_logprobs(z, y.float()),
                lambda: token_logprobs(z[:, :0], y)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        clip_grad_norm([z], 1.0)
    for bad in (lambda: clip_grad_norm([z], -1.0), lambda: clip_grad_norm([z], 1.0, 1.0),
                lambda: clip_grad_norm([y], 1.0), lambda: clip_grad_norm([z], 1.0, out=[]),
                lambda: grad_norm([z], 3.0), lambda: clip_grad_norm([z.to_sparse()], 1.0),
                lambda: clip_grad_norm([z], math.nan)):
        with pytest.raises((ValueError, RuntimeError)):
            bad()
    assert float(clip_grad_norm([], 1.0)) == 0.0


def test_rotary_frequencies():
    from rotary import rotary_frequencies
    inv, f = rotary_frequencies(8, 10000.0)
    assert inv.dtype == torch.float64 and f == 1.0
    assert torch.allclose(inv, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-12)
    assert torch.allclose(rotary_frequencies(8, scaling="linear", factor=4.0)[0], inv / 4, rtol=1e-12)
    b = rotary_frequencies(8, scaling="base", factor=4.0)[0]
    assert torch.allclose(b[[0, -1]], torch.stack([inv[0], inv[-1] / 4]), rtol=1e-12)
    p, f = rotary_frequencies(64, scaling="parts", factor=8.0, trained_length=4096)
    full = rotary_frequencies(64)[0]
    turns = 4096 * full / (2 * math.pi)
    assert torch.allclose(p[turns > 32], full[turns > 32]) and torch.allclose(p[turns < 1], full[turns < 1] / 8)
    assert abs(f - (0.1 * math.log(8) + 1)) < 1e-12
    for bad in (lambda: rotary_frequencies(7), lambda: rotary_frequencies(8, scaling="other"),
                lambda: rotary_frequencies(8, factor=0.5), lambda: rotary_frequencies(8, base=-1.0)):
        with pytest.raises(ValueError):
            bad()


def test_linear_attention_abi_refusals():
    lib = L.load()
    fake = ctypes.c_void_p(4096)  # never dereferenced: every call fails its checks first
    strides = (ctypes.c_int64 * 12)(*[1] * 12)

    def fwd(B=1, T=100, Hk=1, Hv=2, Dk=64, Dv=64, dt=0, gdt=0, p=fake, saved=1 << 40, st=strides):
        return lib.gdn_linatt_fwd(p, p, p, p, p, p, p, p, saved, st, B, T, Hk, Hv, Dk, Dv, 1.0, dt, gdt, None)

    for kw in (dict(B=-1), dict(T=-1), dict(T=0), dict(Hk=0), dict(Hv=0), dict(Dk=0), dict(Dv=0), dict(Hk=2, Hv=3),
               dict(dt=3), dict(gdt=-1), dict(p=None), dict(st=None)):
        assert fwd(**kw) == L.GDN_ERR_INVALID, kw
    for kw in (dict(Dk=257), dict(Dv=300), dict(B=40000, Hv=2), dict(Hk=1, Hv=70000)):
        assert fwd(**kw) == L.GDN_ERR_UNSUPPORTED, kw
    assert fwd(B=0, p=None) == 0
    n = lib.gdn_linatt_saved_bytes(1, 5000, 1, 2, 64, 64)
    assert n > 0 and fwd(T=5000, saved=n - 1) == L.GDN_ERR_WORKSPACE
    assert lib.gdn_linatt_saved_bytes(64, 60, 1, 32, 64, 64) == 64 * 32 * 1024  # one segment: the decays of its chunk
    assert lib.gdn_linatt_saved_bytes(0, 60, 1, 32, 64, 64) == 0

    def bwd(T=100, last=fake, saved=fake, ns=1 << 40, ws=1 << 40, dq=fake):
        return lib.gdn_linatt_bwd(fake, fake, fake, fake, fake, last, saved, ns, fake, fake, dq, fake, fake, fake, fake, fake,
                                  ws, strides, 1, T, 1, 2, 64, 64, 1.0, 0, 0, 0, None)

    assert bwd(last=None) == L.GDN_ERR_INVALID and bwd(dq=None) == L.GDN_ERR_INVALID and bwd(T=0) == L.GDN_ERR_INVALID
    assert bwd(T=5000, saved=None) == L.GDN_ERR_INVALID and bwd(T=5000, ns=n - 1) == L.GDN_ERR_INVALID
    assert bwd(ws=lib.gdn_linatt_bwd_workspace_bytes(1, 100, 1, 2, 64, 64, 0) - 1) == L.GDN_ERR_WORKSPACE
    step = lambda p, Dk: lib.gdn_linatt_step(p, p, p, p, p, p, 1, 1, 1, 1, 2, Dk, 64, 1.0, 0, 0, None)  # noqa: E731
    assert step(None, 64) == L.GDN_ERR_INVALID and step(fake, 0) == L.GDN_ERR_INVALID
    assert step(fake, 300) == L.GDN_ERR_UNSUPPORTED


def test_linear_attention_wrappers_refuse():
    from linear_attention import linear_attention, linear_attention_step
    q, v, g, s = torch.zeros(2, 5, 1, 8), torch.zeros(2, 5, 3, 4), torch.zeros(2, 5, 3), torch.zeros(2, 3, 4, 8)
    for f, a in ((linear_attention, (q, q, v, g, s)), (linear_attention_step, (q[:, 0], q[:, 0], v[:, 0], g[:, 0], s))):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            f(*a)
        for i, bad in ((0, a[0][..., :7]), (1, a[1][:1]), (2, a[2][:1]), (3, a[3][..., :2]), (4, s[:, :2]), (0, a[0].half()),
                       (2, a[2].double()), (3, a[3].int()), (0, a[0][..., 0]), (3, g[0])):
            with pytest.raises(ValueError):
                f(*a[:i], bad, *a[i + 1:])
    with pytest.raises(ValueError, match="divide"):
        linear_attention(torch.zeros(2, 5, 2, 8), torch.zeros(2, 5, 2, 8), v, g, s)
