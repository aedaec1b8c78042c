"""Refusals of MXFP4 weights, and the plain form that the GPU tests compare with (no kernel launches)."""

import ctypes

import pytest
import torch

import gdn_lib as L
import mxfp4_plain as P


def test_abi_refusals():
    lib = L.load()
    fake = ctypes.c_void_p(4096)  # never dereferenced: every call fails its checks first
    quant = lambda N=4, K=40, dt=0, p=fake, c=fake: lib.gdn_mxfp4_quantize(p, c, p, N, K, K, dt, None)  # noqa: E731
    deq = lambda N=4, K=40, dt=0, p=fake, c=fake: lib.gdn_mxfp4_dequantize(c, p, p, N, K, dt, None)  # noqa: E731

    def lin(M=100, K=64, N=128, dt=1, p=fake, c=fake, ld=128, room=1 << 40, f=lib.gdn_mxfp4_linear):
        return f(p, c, p, p, p, room, M, K, N, ld, dt, None)

    back = lambda **kw: lin(f=lib.gdn_mxfp4_linear_bwd, **kw)  # noqa: E731
    odd = ctypes.c_void_p(4100)
    for f in (quant, deq, lin, back):
        for kw in (dict(K=0), dict(N=-1), dict(dt=3), dict(p=None), dict(c=None), dict(c=odd)):
            assert f(**kw) == L.GDN_ERR_INVALID, kw
        for kw in (dict(N=(1 << 24) + 1, **({"ld": 1 << 25} if f in (lin, back) else {})), dict(K=(1 << 18) + 1)):
            assert f(**kw) == L.GDN_ERR_UNSUPPORTED, kw
    assert quant(N=0, p=None) == 0 and deq(N=0, p=None) == 0 and lin(M=0, p=None) == 0 and back(M=0, p=None) == 0
    for f, b in ((lin, 0), (back, 1)):
        assert f(M=-1) == L.GDN_ERR_INVALID and f(N=0) == L.GDN_ERR_INVALID and f(ld=10) == L.GDN_ERR_INVALID
        assert f(M=(1 << 24) + 1) == L.GDN_ERR_UNSUPPORTED
        need = lib.gdn_mxfp4_linear_workspace_bytes(100, 64, 128, 1, 1, b)
        assert need > 0 and f(room=need - 1) == L.GDN_ERR_WORKSPACE
    assert lib.gdn_mxfp4_linear_workspace_bytes(64, 64, 128, 1, 1, 0) == 0
    # a copy of 2^26 elements, and sums in two parts of what they give
    assert lib.gdn_mxfp4_linear_workspace_bytes(1000, 8192, 1 << 20, 1, 1, 0) <= (1 << 27) + 2 * 4 * 1000 * 8192 + (1 << 20)


def test_wrappers_refuse():
    import mxfp4
    w, x = torch.zeros(8, 40), torch.zeros(3, 40)
    q = mxfp4.Weight(torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2, dtype=torch.uint8), 40)
    for f in (lambda: mxfp4.quantize(w), lambda: mxfp4.dequantize(q), lambda: mxfp4.linear(x, q)):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            f()
    for bad in (lambda: mxfp4.quantize(w[0]), lambda: mxfp4.quantize(w.double()), lambda: mxfp4.quantize(w[:, :0]),
                lambda: mxfp4.dequantize(q, torch.float64), lambda: mxfp4.linear(x[:, :39], q), lambda: mxfp4.linear(x.double(), q),
                lambda: mxfp4.linear(x, q._replace(columns=65)), lambda: mxfp4.linear(x, q._replace(codes=q.codes.int())),
                lambda: mxfp4.linear(x, q._replace(scales=q.scales[:7])),
                lambda: mxfp4.linear(x, q._replace(codes=q.codes.t().contiguous().t())),
                lambda: mxfp4.MXFP4Linear.of(torch.nn.Linear(4, 4))):
        with pytest.raises(ValueError):
            bad()


def test_plain_form():
    w = torch.tensor([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9] + [0.0] * 24, [-6.0, 1.0] + [0.0] * 30])
    codes, scales = P.quantize(w)
    assert scales.tolist() == [[127], [127]]
    assert P.values(codes, scales, 9).tolist() == [[0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0, 0.0], [-6.0, 1.0] + [0.0] * 7]
