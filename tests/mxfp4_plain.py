"""MXFP4 in elementary torch operations, written from its definition."""

import torch

E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def quantize(w):
    """(codes, scales) of w [N, K], as bytes."""
    w = torch.nn.functional.pad(w.double(), (0, -w.shape[1] % 32)).unflatten(-1, (-1, 32))
    odd = ~torch.isfinite(w).all(-1)
    w = torch.where(odd[..., None], 0.0, w)
    most = w.abs().amax(-1)
    e = (torch.frexp(most).exponent - 3).clamp_min(-127)
    e = torch.where(most > 0, e, -127)
    m = torch.ldexp(w.abs(), -e[..., None])
    table = torch.tensor(E2M1, dtype=torch.float64, device=w.device)
    gap = (m[..., None] - table).abs()
    even = torch.tensor([0.0, 1.0] * 4, dtype=torch.float64, device=w.device)  # of two as near, the even code
    best = gap.amin(-1, keepdim=True)
    code = torch.where(gap == best, even, 9.0).argmin(-1) | (torch.signbit(w).long() << 3)
    code = torch.where(odd[..., None], 0, code).flatten(-2)
    return (code[:, 0::2] | code[:, 1::2] << 4).to(torch.uint8), torch.where(odd, 255, e + 127).to(torch.uint8)


def values(codes, scales, K):
    """64-bit values [N, K]."""
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    table = torch.tensor(E2M1, dtype=torch.float64, device=codes.device)
    v = table[code & 7] * torch.where(code > 7, -1.0, 1.0).double()
    s = torch.ldexp(torch.ones_like(scales, dtype=torch.float64), scales.int() - 127)
    s = torch.where(scales == 255, float("nan"), s)
    return (v.unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)[:, :K]
