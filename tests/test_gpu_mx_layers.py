"""MXFP4 through the layers, the mixture-of-experts operators and the composed forms."""

import pytest
import torch

import mlxturbo_amd as mq
from mlxturbo_amd import nn, ops, rebit
from mx_helpers import pack, product_tolerance, quantize_ref, values_ref, weights

pytestmark = pytest.mark.gpu

KW = dict(mode="mxfp4")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _check(out, x, v, dtype):
    """out (M, N) against x (M, K) . v (N, K)^T in float64."""
    x = x.double()
    y = x @ v.transpose(-1, -2).contiguous()
    tol = product_tolerance(x, v, y, dtype)
    assert out.dtype == dtype and bool(((out.double() - y).abs() <= tol).all())


# ---- rebit ---------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bias", [False, True])
def test_rebit_keeps_the_float_type(dtype, bias):
    """Affine to MXFP4 and back: scales, biases and outputs of the model's type."""
    g = _gen(1)
    lin = torch.nn.Linear(256, 96, bias=bias, device="cuda", dtype=dtype)
    model = torch.nn.ModuleDict({"lm_head": lin})
    x = _randn(g, 5, 256, dtype=dtype)
    rebit.apply(model, "head=8")
    assert model["lm_head"].scales.dtype == dtype
    rebit.apply(model, "head=mxfp4")
    mid = model["lm_head"]
    v = mid.dequantized_weight()
    assert v.dtype == dtype and mid(x).dtype == dtype
    assert torch.equal(v, mq.dequantize(mid.weight, mid.scales, dtype=dtype, **KW))
    rebit.apply(model, "head=8")
    back = model["lm_head"]
    assert back.mode == "affine" and back.scales.dtype == back.biases.dtype == dtype
    out = back(x)
    assert out.dtype == dtype
    assert back.dequantized_weight().dtype == dtype
    y = mq.quantized_matmul(x, back.weight, back.scales, back.biases, bits=8)
    assert torch.equal(out, y + back.bias if bias else y)


def test_the_float_type_of_a_layer():
    """Given, the bias's, or bfloat16; it follows the module's own conversions."""
    g = _gen(2)
    w, s, _ = weights(g, 48, 64)
    bias = _randn(g, 48, dtype=torch.float16)
    for cls in (nn.QuantizedLinear, nn.QQLinear):
        assert cls(w, s, None, **KW).dequantized_weight().dtype == torch.bfloat16
        assert cls(w, s, None, bias, **KW).dequantized_weight().dtype == torch.float16
        lin = cls(w, s, None, dtype=torch.float32, **KW)
        assert lin.dequantized_weight().dtype == torch.float32
        assert lin.half().dequantized_weight().dtype == torch.float16
        assert set(lin.state_dict()) == {"weight", "scales"}
        f = cls.from_linear(_randn(g, 48, 64, dtype=torch.float16), **KW)
        assert f.dequantized_weight().dtype == torch.float16


# ---- gather_qmm's other forms ----------------------------------------------------

@pytest.mark.parametrize("mode", ["affine", "mxfp4"])
def test_many_experts_and_many_rows(mode):
    """More experts than the pair tables hold and more than 16 rows per pair."""
    g = _gen(3)
    E, N, K, M, P = 2050, 16, 64, 20, 20
    q = mq.quantize(_randn(g, E, N, K, dtype=torch.bfloat16), mode=mode)
    x = _randn(g, P, M, K, dtype=torch.bfloat16)
    rhs = torch.randint(0, E, (P,), generator=g, device="cuda")
    rhs[:3] = torch.tensor([E - 1, 2048, E], device="cuda")
    out = mq.gather_qmm(x, *q[:2], *q[2:], rhs_indices=rhs, mode=mode)
    assert not out[2].any()
    for p in range(P):
        if p != 2:
            e = int(rhs[p])
            v = mq.dequantize(*(t[e] for t in q), mode=mode).double()
            _check(out[p], x[p], v, torch.bfloat16)


def test_many_rows_of_long_weights():
    """More than 16 rows per pair and K beyond the few-pairs kernel."""
    g = _gen(4)
    E, N, K, M = 2, 8, 32 * 9216, 20
    w, s, v = weights(g, E, N, K)
    x = _randn(g, 3, M, K, dtype=torch.bfloat16)
    out = mq.gather_qmm(x, w, s, rhs_indices=torch.tensor([1, 0, 2], device="cuda"), **KW)
    _check(out[0], x[0], v[1], torch.bfloat16)
    _check(out[1], x[1], v[0], torch.bfloat16)
    assert not out[2].any()


def test_many_experts_beyond_the_kernels_ranges():
    """More experts than the pair tables hold, with x of 2 GB and more and K beyond
    the few-pairs kernel: nothing but the composed form takes it."""
    g = _gen(5)
    E, N, K, P = 2050, 1, 32 * 9216, 300
    B = (1 << 31) // (2 * K) + 1
    w = torch.zeros(E, N, K // 8, dtype=torch.int32, device="cuda")
    s = torch.full((E, N, K // 32), 127, dtype=torch.uint8, device="cuda")
    w1, s1, v1 = weights(g, 1, K)
    for e in (7, E - 1):
        w[e], s[e] = w1.view(torch.int32), s1
    x = torch.zeros(B, 1, K, dtype=torch.bfloat16, device="cuda")
    x[B - 1, 0] = _randn(g, K, dtype=torch.bfloat16)
    lhs = torch.full((P,), B - 1, dtype=torch.int32, device="cuda")
    lhs[1] = 0
    rhs = torch.arange(P, dtype=torch.int32, device="cuda")
    rhs[P - 1] = E - 1
    out = mq.gather_qmm(x, w.view(torch.uint32), s, lhs_indices=lhs, rhs_indices=rhs,
                        **KW).reshape(P)
    hit = torch.zeros(P, dtype=torch.bool, device="cuda")
    hit[7] = hit[P - 1] = True
    assert not out[~hit].any()
    _check(out[7].reshape(1, 1), x[B - 1], v1, torch.bfloat16)
    _check(out[P - 1].reshape(1, 1), x[B - 1], v1, torch.bfloat16)


# ---- qqmm -------------------------------------------------------------------------

@pytest.mark.parametrize("M", [3, 20])
def test_qqmm_of_long_rows_at_far_scales(M):
    """float16 x, weights beyond half's range: exact codes at every K, also where K
    is beyond the few-rows kernel (3 rows are composed).  Every product is a whole
    number of halves and their magnitudes sum to less than 2^23, so the float sums
    are exact in any order and the outputs match bit for bit."""
    g = _gen(7)
    N, K = 8, 32 * 9216
    code = torch.randint(0, 16, (N, K), generator=g, device="cuda")
    e = torch.randint(144, 146, (N, K // 32), generator=g, device="cuda")
    v = values_ref(code, e)
    assert float(v.abs().max()) > torch.finfo(torch.float16).max
    x = (torch.randint(-1, 2, (M, K), generator=g, device="cuda") * 2.0 ** -17).half()
    assert torch.equal(values_ref(*quantize_ref(x)), x.double())
    assert bool((x.double().abs() @ v.abs().T.contiguous() < 2 ** 23).all())
    y = x.double() @ v.T.contiguous()
    out = mq.qqmm(x, pack(code), e.to(torch.uint8))
    assert torch.equal(out, y.float().half())


@pytest.mark.parametrize("mode", ["affine", "mxfp4"])
def test_far_batch_indices_of_many_rows(mode):
    """An x batch that does not exist gives zeros, however far off it is (times the
    rows of a pair, these pass 32 bits)."""
    g = _gen(6)
    M, N, K = 20, 16, 64
    q = mq.quantize(_randn(g, 3, N, K, dtype=torch.bfloat16), mode=mode)
    x = _randn(g, 4, M, K, dtype=torch.bfloat16)
    lhs = torch.tensor([3, 1 << 30, 2 ** 31 - 1, -(1 << 30), -(2 ** 31), 4, -1], device="cuda")
    out = mq.gather_qmm(x, *q[:2], *q[2:], lhs_indices=lhs,
                        rhs_indices=torch.ones(7, dtype=torch.int32, device="cuda"), mode=mode)
    v = mq.dequantize(*(t[1] for t in q), mode=mode).double()
    _check(out[0], x[3], v, torch.bfloat16)
    assert not out[1:].any()


# ---- the mixture-of-experts operators ----------------------------------------------

@pytest.mark.parametrize("T", [3, 200])
def test_gather_swiglu_without_tables(T):
    g = _gen(T)
    E, k, H, I = 12, 8, 128, 64
    gate, up = (mq.quantize(_randn(g, E, I, H, dtype=torch.bfloat16)) for _ in range(2))
    x = _randn(g, T, 1, 1, H, dtype=torch.bfloat16)
    idx = torch.randint(0, E, (T, k), generator=g, device="cuda", dtype=torch.int32)
    out = ops.gather_swiglu(x, gate, up, idx, None)
    want = ops.swiglu(mq.gather_qmm(x, *gate, rhs_indices=idx),
                      mq.gather_qmm(x, *up, rhs_indices=idx))
    assert torch.equal(out, want)
    tables = ops.gather_tables(idx, E)
    if tables is not None:
        assert torch.equal(ops.gather_swiglu(x, gate, up, idx, tables), want)


@pytest.mark.parametrize("T", [1, 5, 12, 300])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_moe_operators(T, dtype):
    """gather_swiglu, gather_glu, gather_qmm_combine and moe_layer are their steps,
    bit for bit."""
    g = _gen(T + 40)
    E, k, H, I = 10, 4, 192, 96
    gate, up, down = ((*weights(g, E, *s)[:2], None) for s in ((I, H), (I, H), (H, I)))
    x = _randn(g, T, H, dtype=dtype) * 4
    idx, wts = mq.moe_route(_randn(g, T, E), k)[:2]
    xe = x[:, None, None]
    a, b = (mq.gather_qmm(xe, *bank, rhs_indices=idx, **KW) for bank in (gate, up))
    assert torch.equal(ops.gather_swiglu(xe, gate, up, idx, None, **KW), ops.swiglu(a, b))
    h = ops.gather_glu(xe, *gate, *up, rhs_indices=idx, **KW)
    assert torch.equal(h, (torch.nn.functional.silu(a.float()) * b.float()).to(dtype))
    y = mq.gather_qmm(h, *down, rhs_indices=idx, **KW).reshape(T * k, H)
    want = mq.moe_combine(y, None, wts, T, k)
    assert want.shape == (T, H) and want.dtype == dtype
    assert torch.equal(mq.gather_qmm_combine(h, *down, idx, wts, **KW), want)
    assert torch.equal(ops.moe_layer(x, idx, wts, gate, up, down, **KW), want)
    sgate = torch.rand((T, 1), generator=g, device="cuda").to(dtype)
    shared = _randn(g, T, H, dtype=dtype)
    out = mq.gather_qmm_combine(h, *down, idx, wts, sgate=sgate, shared=shared, **KW)
    assert torch.equal(out, mq.moe_combine(y, None, wts, T, k, sgate, shared))
    with pytest.raises(ValueError, match="together"):
        mq.gather_qmm_combine(h, *down, idx, wts, sgate=sgate, **KW)
