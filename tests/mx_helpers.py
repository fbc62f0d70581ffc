"""MXFP4 in plain torch and 64 bits, for the tests of its operators."""

import torch

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _pow2(p):
    """2^p in float64, p whole and above -1023, from its bits (pow may be off by a
    rounding, which would unmake ties)."""
    return ((p.long() + 1023) << 52).view(torch.float64)


def quantize_ref(v):
    """(codes int64 (..., K), scale bytes int64 (..., K / 32)) of float values,
    by the definition: the group's largest power of two less 2^2, the nearest
    grid value, ties to the even code; a group with a NaN or an infinity is
    byte 255 with zero codes."""
    q = v.double().reshape(*v.shape[:-1], -1, 32)
    bad = ~torch.isfinite(q).all(-1, keepdim=True)
    q = torch.where(bad, 0.0, q)
    top = q.abs().amax(-1, keepdim=True)
    p = torch.frexp(top).exponent.double() - 1 - 2          # floor(log2(top)) - 2
    p = torch.where(top == 0, -127.0, p).clamp_min(-127)
    a = q.abs() / _pow2(p)
    grid = torch.tensor(GRID, dtype=torch.float64, device=q.device)
    d = (a.unsqueeze(-1) - grid).abs()
    best = d.amin(-1, keepdim=True)
    near = d == best                                        # one code, or two at a tie
    even = near & (torch.arange(8, device=q.device) % 2 == 0)
    pick = torch.where(even.any(-1, keepdim=True), even, near)
    code = pick.int().argmax(-1) + 8 * torch.signbit(q)
    code = torch.where(bad, 0, code)
    e = torch.where(bad.squeeze(-1), 255, (p.squeeze(-1) + 127).long())
    return code.reshape(v.shape), e


def values_ref(code, e):
    """What codes and scale bytes stand for, in float64."""
    grid = torch.tensor(GRID + tuple(-g for g in GRID), dtype=torch.float64, device=code.device)
    s = torch.where(e == 255, float("nan"), _pow2(e.long() - 127))
    v = grid[code].reshape(*e.shape, 32) * s.unsqueeze(-1)
    return v.reshape(code.shape)


def pack(code):
    """Codes -> uint32 words, low bits first."""
    b = (code[..., 0::2] | (code[..., 1::2] << 4)).to(torch.uint8).contiguous()
    return b.view(torch.int32).view(torch.uint32)


def unpack(w):
    b = w.contiguous().view(torch.int32).view(torch.uint8).long()
    return torch.stack([b & 15, b >> 4], -1).reshape(*b.shape[:-1], -1)


def weights(g, *shape, device="cuda", scale=0.02):
    """Random MXFP4 weights: (words, scale bytes, their values in float64)."""
    v = torch.randn(shape, generator=g, device=device) * scale
    code, e = quantize_ref(v)
    return pack(code), e.to(torch.uint8), values_ref(code, e)


def product_tolerance(x, v, y, dtype):
    """How far a product x . v^T (float64, y the sums) rounded to dtype may be
    from y, elementwise: half a step of the type (relative eps / 2, or half its
    smallest step) plus the float sum's error in any order, at most 2^-23 of
    the sum of magnitudes per addition (an MFMA's additions need not round to
    nearest), itself rounded once more."""
    eps = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * eps
    mag = x.abs() @ v.abs().transpose(-1, -2)
    acc = (x.shape[-1] + 16) * 2.0 ** -23 * mag
    return eps * y.abs() + tiny + acc * (1 + eps)
