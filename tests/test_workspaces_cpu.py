"""The workspace that the queries grant is what the calls ask for, whatever the operands' layout (no kernel launches)."""

import re

import pytest
import torch

import gdn_lib as L

FAR = 4096 * 2048  # elements: the last hidden states of sequences of 4096 tokens of 2048 channels


def rows(n, cols, dtype, stride):
    """A tensor of such a layout, without memory."""
    return torch.empty_strided((n, cols), (stride, 1), dtype=dtype, device="meta")


def needed(call):
    """What a call without room asks for."""
    assert call() == L.GDN_ERR_WORKSPACE
    return int(re.search(rb"(\d+) are needed", L.load().gdn_last_error()).group(1))


def layouts(H):
    """(row stride in elements, the address's offset in bytes): as they should be, off 16 bytes, odd, and far apart."""
    return ((H, 0), (H + 8, 0), (H, 2), (H + 1, 0), (FAR, 0), (FAR + 4, 0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("N,H,V", [(1, 64, 100), (8, 2048, 32000), (64, 128, 3000), (100, 256, 70000), (130, 64, 7), (400, 64, 32000),
                                   (400, 128, 3000), (400, 2048, 300), (500, 64, 32000), (511, 4096, 100), (512, 64, 5000),
                                   (700, 70, 20000), (2047, 64, 1000), (2500, 128, 9000)])
def test_loss(N, H, V, dtype):
    """x and the weight lie in any two ways: the room that the wrapper asks for is enough for both calls."""
    lib, code = L.load(), L.DTYPE_CODE[dtype]
    fake = 1 << 20  # never dereferenced: the calls fail for want of room
    for xs, xo in layouts(H):
        for ws, wo in layouts(H):
            x, w = rows(N, H, dtype, xs), rows(V, H, dtype, ws)
            well = L.rows_lie_well(x, w) and not xo and not wo
            xs, ws = L.row_stride(x), L.row_stride(w)
            room = lib.gdn_linear_loss_workspace_bytes(N, H, V, code, well, 0, 0)
            fwd = needed(lambda: lib.gdn_linear_loss_fwd(fake + xo, fake + wo, fake, fake, fake, fake, fake, fake, 0, N, H, V, xs, ws,
                                                         -100, 0, code, None))
            assert fwd <= room, (xs, xo, ws, wo, fwd, room)
            for dx, dw in ((fake, None), (None, fake), (fake, fake)):
                room = lib.gdn_linear_loss_workspace_bytes(N, H, V, code, well, dx is not None, dw is not None)
                bwd = needed(lambda: lib.gdn_linear_loss_bwd(fake + xo, fake + wo, fake, fake, fake, 1, None, dx, dw, fake, 0, N, H, V,
                                                             xs, ws, -100, code, None))
                assert bwd <= room, (xs, xo, ws, wo, dx, dw, bwd, room)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,K,N", [(1, 64, 64), (65, 64, 128), (100, 2048, 8192), (65, 2048, 8192), (300, 70, 1000), (1000, 128, 70),
                                   (70, 256, 300000)])
def test_linear(M, K, N, dtype):
    lib, code = L.load(), L.DTYPE_CODE[dtype]
    fake = 1 << 20
    for back, cols in ((0, K), (1, N)):
        for stride, off in layouts(cols):
            x = rows(M, cols, dtype, stride)
            well, stride = L.rows_lie_well(x) and not off, L.row_stride(x)
            room = lib.gdn_mxfp4_linear_workspace_bytes(M, K, N, code, well, back)
            if not back and M <= 64:
                assert room == 0
                continue
            call = lib.gdn_mxfp4_linear_bwd if back else lib.gdn_mxfp4_linear
            need = needed(lambda: call(fake + off, fake, fake, fake, fake, 0, M, K, N, stride, code, None))
            assert need <= room, (back, stride, off, need, room)
