"""MXFP4 products whose float sums are exact, so the outputs have to match bit for
bit, and products at the ends of the scales' range."""

import pytest
import torch

import mlxturbo_amd as mq
from mx_helpers import pack, product_tolerance, quantize_ref, values_ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
KW = dict(mode="mxfp4")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randint(g, lo, hi, *shape):
    return torch.randint(lo, hi, shape, generator=g, device="cuda")


def _weights(g, *shape):
    """Random codes under scales of 1/2, 1 and 2: (words, scale bytes, values in
    float64).  Values are multiples of 1/4 of at most 12, exact in both types."""
    code = _randint(g, 0, 16, *shape)
    e = _randint(g, 126, 129, *shape[:-1], shape[-1] // 32)
    return pack(code), e.to(torch.uint8), values_ref(code, e)


def _activations(g, M, K, qq, dtype):
    """Whole numbers up to 2, or, qq, values that the format holds exactly: of
    random codes under scales of 1/2, 1 and 2, a 6 in every group so that the
    quantizer finds the same scale."""
    if not qq:
        return _randint(g, -2, 3, M, K).to(dtype)
    code = _randint(g, 0, 16, M, K)
    code[:, ::32] = 7
    x = values_ref(code, _randint(g, 126, 129, M, K // 32))
    assert torch.equal(values_ref(*quantize_ref(x)), x)
    return x.to(dtype)


def _exact(x, v, dtype):
    """x . v^T rounded once.  x is of multiples of 1/4 and v too, so any partial sum
    is a multiple of 1/16; the sum of magnitudes below 2^20 makes every one of them
    exact in float's 24 bits, in whatever order they are added."""
    x = x.double()
    assert bool((x.abs() @ v.abs().transpose(-1, -2).contiguous() < 2 ** 20).all())
    y = x @ v.transpose(-1, -2).contiguous()
    return y.float().to(dtype)


# up to 8, 16 rows (skinny), 17 to 64 (the K splits of a 64-row tile), tall tiles;
# K in whole 512s, in whole groups and steps alone
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K", [17408, 17440, 13696, 5152, 800])
@pytest.mark.parametrize("M", [1, 8, 13, 17, 45, 64, 300])
@pytest.mark.parametrize("qq", [False, True])
def test_products_bit_for_bit(M, K, dtype, qq):
    g = _gen(M + K)
    N = 201
    w, s, v = _weights(g, N, K)
    x = _activations(g, M, K, qq, dtype)
    out = mq.qqmm(x, w, s) if qq else mq.quantized_matmul(x, w, s, **KW)
    assert torch.equal(out, _exact(x, v, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K", [17408, 5152, 768])
@pytest.mark.parametrize("P,E", [(5, 3), (200, 4), (300, 50), (1000, 3)])
def test_gather_bit_for_bit(P, E, K, dtype):
    g = _gen(P + K)
    N = 70
    w, s, v = _weights(g, E, N, K)
    x = _activations(g, P, K, False, dtype)
    rhs = _randint(g, 0, E, P).int()
    out = mq.gather_qmm(x[:, None], w, s, rhs_indices=rhs, **KW).reshape(P, N)
    for e in range(E):
        rows = (rhs == e).nonzero().flatten()
        assert torch.equal(out[rows], _exact(x[rows], v[e], dtype))


# (type, scale bytes, power of two of x): half-subnormal weights, weights that round
# to half's smallest steps, both ends of bf16's range
RANGES = [(torch.float16, 103, 114, 6), (torch.float16, 95, 106, 12),
          (torch.float16, 134, 141, -8), (torch.bfloat16, 0, 4, 100),
          (torch.bfloat16, 1, 40, 90), (torch.bfloat16, 215, 253, -110)]


@pytest.mark.parametrize("dtype,lo,hi,p", RANGES)
@pytest.mark.parametrize("M", [1, 12, 40, 300])
@pytest.mark.parametrize("K", [512, 160])
def test_products_at_far_scales(M, K, dtype, lo, hi, p):
    """The sums run over T(code * 2^(e - 127)), subnormal ones among them."""
    g = _gen(M + K + lo)
    N = 65
    code = _randint(g, 0, 16, N, K)
    e = _randint(g, lo, hi, N, K // 32)
    w, s = pack(code), e.to(torch.uint8)
    v = values_ref(code, e).float().to(dtype).double()      # float holds the values exactly
    assert v.isfinite().all()
    x = (torch.randn((M, K), generator=g, device="cuda").double() * 2.0 ** p).to(dtype)
    y = x.double() @ v.T.contiguous()
    assert float(y.abs().max()) < torch.finfo(dtype).max
    tol = product_tolerance(x.double(), v, y, dtype)
    out = mq.quantized_matmul(x, w, s, **KW)
    assert bool(((out.double() - y).abs() <= tol).all())
    out = mq.gather_qmm(x[None], w[None], s[None], rhs_indices=torch.zeros(1, device="cuda").int(),
                        **KW)[0]
    assert bool(((out.double() - y).abs() <= tol).all())


# (type, scale bytes of w, power of two of x)
QQ_RANGES = [(torch.float16, 95, 110, 12), (torch.float16, 140, 148, -14),
             (torch.bfloat16, 0, 20, 100), (torch.bfloat16, 235, 255, -115),
             (torch.bfloat16, 60, 70, 60)]


@pytest.mark.parametrize("dtype,lo,hi,p", QQ_RANGES)
@pytest.mark.parametrize("M", [1, 12, 40, 300])
@pytest.mark.parametrize("K", [512, 160])
def test_qqmm_at_far_scales(M, K, dtype, lo, hi, p):
    """Both sides enter with their scales, so a weight that T does not hold is
    multiplied as it is."""
    g = _gen(M + K + lo + 1)
    N = 65
    code = _randint(g, 0, 16, N, K)
    e = _randint(g, lo, hi, N, K // 32)
    v = values_ref(code, e)
    x = (torch.randn((M, K), generator=g, device="cuda").double() * 2.0 ** p).to(dtype)
    xv = values_ref(*quantize_ref(x))
    y = xv @ v.T.contiguous()
    assert float(y.abs().max()) < torch.finfo(dtype).max
    tol = product_tolerance(xv, v, y, dtype)
    out = mq.qqmm(x, pack(code), e.to(torch.uint8))
    assert bool(((out.double() - y).abs() <= tol).all())
