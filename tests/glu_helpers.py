"""The gated feed-forward block over affine weights in 64 bits, for its tests, with
how far the kernels' results may be from it."""

import math

import torch

ACTS = ("silu", "gelu_tanh")


def bank(g, N, K, gs, bits, dtype, device="cuda", scale=0.02):
    """Random affine weights: (words, scales, biases) and their values in float64:
    scale * code + bias, rounded to float (the sum) and to dtype."""
    code = torch.randint(0, 2 ** bits, (N, K), generator=g, device=device)
    s = ((0.5 + torch.rand((N, K // gs), generator=g, device=device)) * scale * 4
         / 2 ** bits).to(dtype)
    b = (-2 * scale + scale * torch.rand((N, K // gs), generator=g, device=device)).to(dtype)
    return (pack(code, bits), s, b), values(code, s, b, gs)


def pack(code, bits):
    """Codes -> uint32 words, low bits first."""
    b = code.to(torch.uint8)
    if bits == 4:
        b = b[:, 0::2] | (b[:, 1::2] << 4)
    return b.contiguous().view(torch.int32).view(torch.uint32)


def values(code, s, b, gs):
    sd, bd = (t.double().repeat_interleave(gs, dim=1) for t in (s, b))
    return (sd * code.double() + bd).float().to(s.dtype).double()


def activation(g, act):
    """act(g) and its derivative, in float64."""
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * (1 - s)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 0.134145 * g * g)


def _sum_error(x, w):
    """What the float sum of x . w^T over exact products, in any order, may be off:
    at most 2^-23 of the sum of magnitudes per addition (an MFMA's additions need not
    round to nearest)."""
    return (x.shape[-1] + 16) * 2.0 ** -23 * (x.abs() @ w.abs().T)


def _round(y, dtype):
    """Half a step of the type at y, or half its smallest step."""
    f = torch.finfo(dtype)
    return (f.eps / 2) * y.abs() + f.smallest_normal * f.eps / 2


def glu_ref(x, wg, wu, act, dtype):
    """h in float64 and how far a kernel's may be: its sums' error through the
    activation (|act'| < 1.13 for both), the activation's own few float roundings (8,
    and expf within two units of the last place, times an argument's error of 2^-22 of
    the exponent, which |act| scales by |g| at most), the product and the last rounding."""
    x = x.double()
    g, u = x @ wg.T, x @ wu.T
    a, _ = activation(g, act)
    h = a * u
    eg, eu = _sum_error(x, wg), _sum_error(x, wu)
    ea = 1.13 * eg + (16 + 4 * g.abs()) * 2.0 ** -23 * a.abs() + 2.0 ** -126
    off = ea * (u.abs() + eu) + a.abs() * eu
    return h, _round(h.abs() + off, dtype) + off


def glu_grad_ref(x, d, wg, wu, act, dtype):
    """dL/dx for dL/dh = d in float64 and how far a kernel's may be: the errors of g
    and u (|act''| < 1.2 for both), of the activation in float, the rounding of dg and
    du to dtype, the float sum over both halves, and the last rounding."""
    x, d = x.double(), d.double()
    g, u = x @ wg.T, x @ wu.T
    a, da = activation(g, act)
    eg, eu = _sum_error(x, wg), _sum_error(x, wu)
    rel = (16 + 4 * g.abs()) * 2.0 ** -23
    ea, eda = 1.13 * eg + rel * a.abs() + 2.0 ** -126, 1.2 * eg + rel * 1.2
    dg, du = d * u * da, d * a
    edg = d.abs() * ((u.abs() + eu) * eda + eu * da.abs())
    edu = d.abs() * ea
    edg, edu = edg + _round(dg.abs() + edg, dtype), edu + _round(du.abs() + edu, dtype)
    dx = dg @ wg + du @ wu
    mag = (dg.abs() + edg) @ wg.abs() + (du.abs() + edu) @ wu.abs()
    off = edg @ wg.abs() + edu @ wu.abs() + (2 * wg.shape[0] + 16) * 2.0 ** -23 * mag
    return dx, off + _round(dx.abs() + off, dtype)


def matmul_ref(x, w, dtype):
    """x . w^T in float64 and how far a kernel's may be."""
    x = x.double()
    y, off = x @ w.T, _sum_error(x, w)
    return y, off + _round(y.abs() + off, dtype)


def check(got, want, tol, what=""):
    got = got.double()
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), (
        f"{what}: {int(bad.sum())} of {bad.numel()} off, worst "
        f"{float(((got - want).abs() / tol).nan_to_num(float('inf')).max()):.3g} of the tolerance, "
        f"first at {bad.nonzero()[0].tolist()}")
