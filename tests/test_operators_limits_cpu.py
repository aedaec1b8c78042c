"""Sizes that no launch can take are refused by the operators' checks, before anything runs (no kernel launches)."""

import ctypes

import gdn_lib as L


def test_logprobs_pieces():
    """A workgroup of 256 threads for each piece, less than 2^32 threads in all."""
    lib = L.load()

    def fwd(outer, inner, V):
        return lib.gdn_logprobs_fwd(*[None] * 8, 0, outer, inner, V, 0, V, -100, 0, 0, None)

    def bwd(outer, inner, V):
        return lib.gdn_logprobs_bwd(*[None] * 7, outer, inner, V, 0, V, -100, 0, None)

    for call in (fwd, bwd):
        for size in ((1 << 24, 1, 10), (1, 1 << 24, 10), (1 << 23, 1, 8193), (1 << 12, 1 << 12, 10), (1, 1 << 40, 10)):
            assert call(*size) == L.GDN_ERR_UNSUPPORTED, size
        # the largest that can run fail at the next check, their null pointers
        for size in (((1 << 24) - 1, 1, 10), (1, (1 << 23) - 1, 8193)):
            assert call(*size) == L.GDN_ERR_INVALID, size


def test_linear_attention_elements():
    lib = L.load()
    strides = (ctypes.c_int64 * 12)()

    def fwd(B, T, Hv, D):
        return lib.gdn_linatt_fwd(*[None] * 8, 0, strides, B, T, 1, Hv, D, D, 1.0, 0, 0, None)

    for size in ((60000, (1 << 31) - 1, 1, 256), (1 << 8, 1 << 30, 2, 1), (2, 1 << 30, 1, 256)):
        assert fwd(*size) == L.GDN_ERR_UNSUPPORTED, size
    assert fwd(1, 1 << 30, 1, 256) == L.GDN_ERR_INVALID  # null pointers


def test_steps_of_many_sequences():
    """A step's sequences and heads are counted apart: 4096 sequences of 32 heads pass (and fail for their null pointers)."""
    lib = L.load()
    step = lambda B, Hv: lib.gdn_linatt_step(*[None] * 6, 1, 1, B, 1, Hv, 64, 64, 1.0, 0, 0, None)  # noqa: E731
    assert step(4096, 32) == L.GDN_ERR_INVALID and step(65535, 65535) == L.GDN_ERR_INVALID
    assert step(65536, 1) == L.GDN_ERR_UNSUPPORTED and step(1, 65536) == L.GDN_ERR_UNSUPPORTED
