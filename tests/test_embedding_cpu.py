"""Refusals of the embedding, and its module on the CPU (no kernel launches)."""

import ctypes

import pytest
import torch

import gdn_lib as L


def test_abi_refusals():
    lib = L.load()
    fake = ctypes.c_void_p(4096)  # never dereferenced: every call fails its checks first
    fwd = lambda N=4, V=9, H=8, dt=0, p=fake: lib.gdn_embedding_fwd(p, p, p, N, V, H, H, 1.0, dt, None)  # noqa: E731
    bwd = lambda N=4, V=9, H=8, dt=0, p=fake, room=1 << 40: lib.gdn_embedding_bwd(  # noqa: E731
        p, p, p, p, room, N, V, H, H, -1, 1.0, dt, None)
    for f in (fwd, bwd):
        for kw in (dict(N=-1), dict(V=0), dict(H=0), dict(dt=3), dict(p=None)):
            assert f(**kw) == L.GDN_ERR_INVALID, kw
        for kw in (dict(N=(1 << 26) + 1), dict(V=1 << 22), dict(H=(1 << 20) + 1)):
            assert f(**kw) == L.GDN_ERR_UNSUPPORTED, kw
    assert fwd(N=0, p=None) == 0
    assert bwd(room=lib.gdn_embedding_bwd_workspace_bytes(4, 9, 8) - 1) == L.GDN_ERR_WORKSPACE
    assert lib.gdn_embedding_bwd_workspace_bytes(-1, 9, 8) == 0


def test_wrapper_refuses():
    from embedding import Embedding, embedding
    ids, w = torch.zeros(3, dtype=torch.int64), torch.zeros(10, 4)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        embedding(ids, w)
    for bad in (lambda: embedding(ids.float(), w), lambda: embedding(ids, w[0]), lambda: embedding(ids, w.double()),
                lambda: embedding(ids, w[:0]), lambda: embedding(ids, w, padding_idx=10), lambda: embedding(ids, w, padding_idx=-1),
                lambda: Embedding(4, 4, sparse=True), lambda: Embedding(4, 4, max_norm=1.0)):
        with pytest.raises(ValueError):
            bad()


def test_module_on_the_cpu():
    from embedding import Embedding
    m = Embedding(10, 4, 2, scale=2.0)
    ids = torch.tensor([[1, 2], [2, 9]])
    assert torch.equal(m(ids), torch.nn.functional.embedding(ids, m.weight, 2) * 2)
