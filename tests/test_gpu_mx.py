"""The MXFP4 operators on the GPU against their definitions in 64 bits."""

import threading

import pytest
import torch

import mlxturbo_amd as mq
from mlxturbo_amd import nn, ops, rebit
from mx_helpers import (pack, product_tolerance, quantize_ref, unpack, values_ref,
                        weights)

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
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
    off = (out.double() - y).abs()
    assert out.dtype == dtype and bool((off <= tol).all()), (
        f"off by {float((off / tol).max()):.3g} tolerances")


# ---- quantize, dequantize ------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES + [torch.float32])
@pytest.mark.parametrize("N,K", [(1, 32), (3, 96), (257, 160), (64, 4096)])
def test_quantize_bits(dtype, N, K):
    g = _gen(1)
    v = _randn(g, N, K, dtype=dtype)
    # group magnitudes over the type's range
    info = torch.finfo(dtype)
    lo = -140 if dtype != torch.float16 else -24
    hi = 125 if dtype != torch.float16 else 13
    p = torch.randint(lo, hi, (N, K // 32, 1), generator=g, device="cuda").double()
    v = (v.double().reshape(N, -1, 32).clamp(-3, 3) * torch.pow(2.0, p)).clamp(
        info.min, info.max).reshape(N, K).to(dtype)
    wq, s = mq.quantize(v, **KW)
    code, e = quantize_ref(v)
    assert wq.dtype == torch.uint32 and s.dtype == torch.uint8
    assert torch.equal(s.long(), e)
    assert torch.equal(unpack(wq), code)


@pytest.mark.parametrize("dtype", DTYPES + [torch.float32])
def test_quantize_ties_and_ends(dtype):
    # every multiple of 1/16 up to 8 under scale 1 (7.99 sets it), ties included
    k = torch.arange(0, 128, device="cuda").float() / 16
    v = torch.stack([k, -k]).reshape(-1)[:248].reshape(8, 31)
    v = torch.cat([torch.full((8, 1), 7.5, device="cuda"), v], 1)
    rest = torch.zeros(8, 32, device="cuda")
    rest[0] = -0.0
    rest[1, 5] = float("nan")
    rest[2, 31] = float("inf")
    rest[3, 0] = -float("inf")
    rest[4, 7] = torch.finfo(dtype).max
    rest[5, 7] = torch.finfo(dtype).smallest_normal
    rest[6, 7] = torch.finfo(dtype).smallest_normal / 4     # subnormal
    rest[7, 3:5] = torch.tensor([1.0, 1e-30], device="cuda")
    v = torch.cat([v, rest], 1).to(dtype)
    wq, s = mq.quantize(v, **KW)
    code, e = quantize_ref(v)
    assert torch.equal(s.long(), e) and torch.equal(unpack(wq), code)
    assert (s[1:4, 1] == 255).all() and not unpack(wq)[1:4, 32:].any()


@pytest.mark.parametrize("dtype", DTYPES + [torch.float32])
def test_dequantize_every_code_and_scale(dtype):
    code = torch.arange(16, device="cuda").repeat(256, 2)    # (256, 32)
    e = torch.arange(256, device="cuda")[:, None]
    out = mq.dequantize(pack(code), e.to(torch.uint8), dtype=dtype, **KW)
    want = values_ref(code, e).float().to(dtype)             # float32 holds all but none is lost
    assert out.dtype == dtype
    assert torch.equal(out.isnan(), want.isnan())
    ok = ~want.isnan()
    assert torch.equal(out[ok], want[ok])
    assert torch.equal(torch.signbit(out[ok]), torch.signbit(want[ok]))


def test_format_shapes_and_strides():
    g = _gen(2)
    v = _randn(g, 4, 6, 128, dtype=torch.bfloat16)
    wq, s = mq.quantize(v.transpose(0, 1), **KW)
    assert wq.shape == (6, 4, 16) and s.shape == (6, 4, 4)
    a, b = mq.quantize(v.transpose(0, 1).contiguous(), **KW)
    assert torch.equal(wq.view(torch.int32), a.view(torch.int32)) and torch.equal(s, b)
    flat = torch.empty(6 * 4 * 128 + 1, device="cuda", dtype=torch.bfloat16)[1:]   # 2-byte base
    flat.copy_(v.transpose(0, 1).reshape(-1))
    c, d = mq.quantize(flat.reshape(6, 4, 128), **KW)
    assert torch.equal(c.view(torch.int32), a.view(torch.int32)) and torch.equal(d, b)
    full = mq.dequantize(a, b, **KW)
    assert full.dtype == torch.bfloat16 and full.shape == (6, 4, 128)
    part = mq.dequantize(a.view(torch.int32)[:, 1:3].view(torch.uint32), b[:, 1:3], **KW)
    assert torch.equal(part, full[:, 1:3])
    e8 = mq.dequantize(a, b.view(torch.float8_e8m0fnu), **KW)
    assert torch.equal(e8, full)
    wq, s = mq.quantize(v[0, 0], **KW)                       # one row without a leading dim
    assert wq.shape == (16,) and torch.equal(mq.dequantize(wq, s, **KW),
                                             mq.dequantize(*mq.quantize(v[:1, 0], **KW), **KW)[0])


# ---- products ------------------------------------------------------------------

SHAPES = [(1, 1, 32), (1, 16, 128), (2, 17, 96), (5, 250, 160), (16, 33, 1056), (17, 64, 512),
          (31, 100, 544), (33, 48, 2080), (64, 30, 256), (65, 257, 320), (130, 515, 1152),
          (1, 12000, 352), (300, 260, 64), (3, 10300, 64), (48, 10250, 96), (7, 40, 17408),
          (513, 640, 832), (192, 256, 2048), (200, 300, 17440), (1000, 128, 5152), (70, 70, 32),
          (2049, 33, 96), (129, 1030, 3584)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_quantized_matmul(M, N, K, dtype):
    g = _gen(M + N + K)
    w, s, v = weights(g, N, K)
    x = _randn(g, M, K, dtype=dtype)
    _check(mq.quantized_matmul(x, w, s, **KW), x, v, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_qqmm(M, N, K, dtype):
    g = _gen(M + N + K + 1)
    w, s, v = weights(g, N, K)
    x = _randn(g, M, K, dtype=dtype)
    _check(mq.qqmm(x, w, s), values_ref(*quantize_ref(x)), v, dtype)


@pytest.mark.parametrize("N,K", [(100, 1056), (10300, 160), (90, 9248)])
def test_rows_do_not_depend_on_the_row_count(N, K):
    g = _gen(3)
    w, s, _ = weights(g, N, K)
    x = _randn(g, 32, K, dtype=torch.bfloat16)
    for f in (lambda a: mq.quantized_matmul(a, w, s, **KW), lambda a: mq.qqmm(a, w, s)):
        full = f(x[:16])
        for m in (1, 2, 8, 9):
            assert torch.equal(f(x[:m]), full[:m])
        with mq.row_identity():
            full = f(x)
            for m in (1, 8, 16, 17, 31):
                assert torch.equal(f(x[:m]), full[:m])


def test_product_strides_and_leading_dims():
    g = _gen(4)
    w, s, v = weights(g, 70, 192)
    x = _randn(g, 3, 5, 192, dtype=torch.bfloat16)
    want = mq.quantized_matmul(x.reshape(15, 192), w, s, **KW)
    _check(want, x.reshape(15, 192), v, torch.bfloat16)
    assert torch.equal(mq.quantized_matmul(x, w, s, **KW), want.reshape(3, 5, 70))
    xt = x.transpose(0, 1)                                   # not contiguous
    assert torch.equal(mq.quantized_matmul(xt, w, s, **KW), want.reshape(3, 5, 70).transpose(0, 1))
    flat = torch.empty(15 * 192 + 1, dtype=torch.bfloat16, device="cuda")[1:]
    flat.copy_(x.reshape(-1))
    assert torch.equal(mq.quantized_matmul(flat.reshape(15, 192), w, s, **KW), want)
    # a slice of a bank's rows: scales that start anywhere
    w2, s2 = w.view(torch.int32)[3:].view(torch.uint32), s[3:]
    assert torch.equal(mq.quantized_matmul(x, w2, s2, **KW), want.reshape(3, 5, 70)[..., 3:])
    assert torch.equal(mq.qqmm(x, w2, s2), mq.qqmm(x, w, s)[..., 3:])
    # float32 activations and transpose=False run as dequantize and a GEMM
    xf = x.float()
    out = mq.quantized_matmul(xf, w, s, **KW)
    assert out.dtype == torch.float32
    assert torch.allclose(out.double(), xf.double() @ v.T, rtol=0, atol=1e-4)
    wt, st, vt = weights(g, 48, 64)                          # [K=48, N=64]
    xs = _randn(g, 4, 48, dtype=torch.bfloat16)
    out = mq.quantized_matmul(xs, wt, st, transpose=False, **KW)
    _check(out, xs, vt.T.contiguous(), torch.bfloat16)


@pytest.mark.parametrize("M", [1, 5, 40, 300])
def test_infinities_and_nans_stay_where_they_belong(M):
    g = _gen(5)
    N, K = 90, 160                                           # five groups: a ragged last step
    w, s, v = weights(g, N, K)
    x = _randn(g, M, K, dtype=torch.bfloat16)
    clean = mq.quantized_matmul(x, w, s, **KW)
    clean_q = mq.qqmm(x, w, s)
    s2 = s.clone()
    s2[17, 4] = 255                                          # NaN group of the last weight group
    for f, c in ((lambda a, b: mq.quantized_matmul(a, w, b, **KW), clean),
                 (lambda a, b: mq.qqmm(a, w, b), clean_q)):
        out = f(x, s2)
        assert out[:, 17].isnan().all()
        keep = [n for n in range(N) if n != 17]
        assert torch.equal(out[:, keep], c[:, keep])
        bad = x.clone()
        bad[M - 1, 3] = float("inf")
        out = f(bad, s)
        assert not out[M - 1].isfinite().any()
        assert torch.equal(out[:M - 1], c[:M - 1])
    # inf * w is inf with w's sign, inf * 0 NaN, elsewhere untouched: no padding adds NaNs
    bad = x.clone()
    bad[0, 3] = float("inf")
    col = v[:, 3]
    out = mq.quantized_matmul(bad, w, s, **KW)[0]
    assert torch.equal(out.isnan(), col == 0)
    assert torch.equal(out[col != 0], torch.sign(col[col != 0]).to(out.dtype) * float("inf"))


@pytest.mark.parametrize("dtype", DTYPES)
def test_scales_over_the_whole_range(dtype):
    """Groups whose scales lie far apart: sums are dominated by the largest,
    and the small ones are not flushed."""
    g = _gen(6)
    N, K = 33, 128
    code = torch.randint(0, 16, (N, K), generator=g, device="cuda")
    lo, hi = (115, 140) if dtype == torch.float16 else (60, 190)
    e = torch.randint(lo, hi, (N, K // 32), generator=g, device="cuda")
    w, s, v = pack(code), e.to(torch.uint8), values_ref(code, e)
    for M in (4, 80):
        x = _randn(g, M, K, dtype=dtype)
        x[:, :64] = 0 if dtype == torch.float16 else x[:, :64] * 2.0 ** -60
        y = x.double() @ v.T
        out = mq.quantized_matmul(x, w, s, **KW)
        fits = y.abs() < torch.finfo(dtype).max
        tol = product_tolerance(x.double(), v, y, dtype)
        assert bool(((out.double() - y).abs() <= tol)[fits].all())


# ---- gather --------------------------------------------------------------------

def _gather_ref(x, v, lhs, rhs):
    """x (B, M, K), v (E, N, K): (P, M, N) sums in float64 and tolerances."""
    ok = (rhs >= 0) & (rhs < v.shape[0]) & (lhs >= 0) & (lhs < x.shape[0])
    xs = x[lhs.clamp(0, x.shape[0] - 1).long()].double()
    vs = v[rhs.clamp(0, v.shape[0] - 1).long()]
    y = torch.matmul(xs, vs.transpose(1, 2).contiguous())
    tol = product_tolerance(xs, vs.contiguous(), y, x.dtype)
    return y * ok[:, None, None], tol, ok


def _check_gather(out, x, v, lhs, rhs):
    y, tol, ok = _gather_ref(x, v, lhs, rhs)
    out = out.reshape(y.shape)
    assert bool(((out.double() - y).abs() <= tol).all())
    assert not out[~ok].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,E,N,K,zipf", [
    (1, 1, 1, 16, 32, False), (1, 8, 64, 48, 256, False), (3, 2, 5, 33, 160, False),
    (8, 8, 16, 130, 352, True), (32, 8, 7, 64, 96, True), (40, 8, 64, 50, 128, True),
    (301, 4, 30, 257, 320, False), (700, 3, 9, 96, 544, True), (256, 4, 500, 64, 64, False),
    (1500, 1, 3, 300, 192, False)])
def test_gather_qmm(T, k, E, N, K, zipf, dtype):
    g = _gen(T + k + E + N + K)
    w, s, v = weights(g, E, N, K)
    x = _randn(g, T, 1, 1, K, dtype=dtype)
    p = torch.arange(1, E + 1, device="cuda").float() ** (-1.3 if zipf else 0)
    idx = torch.multinomial(p.expand(T, E), k, replacement=k > E, generator=g).int()
    out = mq.gather_qmm(x, w, s, rhs_indices=idx, **KW)
    assert out.shape == (T, k, 1, N) and out.dtype == dtype
    lhs = torch.arange(T, device="cuda").repeat_interleave(k)
    _check_gather(out, x.reshape(T, 1, K), v, lhs, idx.reshape(-1))


@pytest.mark.parametrize("P,B,M", [(5, 3, 1), (6, 3, 4), (9, 4, 16), (40, 8, 3), (300, 50, 1),
                                   (200, 20, 7), (80, 9, 20)])
def test_gather_indices_rows_and_invalid_pairs(P, B, M):
    g = _gen(P + B + M)
    E, N, K = 6, 70, 160
    w, s, v = weights(g, E, N, K)
    x = _randn(g, B, M, K, dtype=torch.bfloat16)
    rhs = torch.randint(-1, E + 1, (P,), generator=g, device="cuda")
    lhs = torch.randint(0, B, (P,), generator=g, device="cuda")
    if P > 8:
        lhs[2], lhs[5] = -1, B
    out = mq.gather_qmm(x, w, s, lhs_indices=lhs, rhs_indices=rhs, **KW)
    assert out.shape == (P, M, N)
    _check_gather(out, x, v, lhs, rhs)
    # the same expert for every pair, and sorted pairs
    one = torch.full((P,), 4, device="cuda")
    _check_gather(mq.gather_qmm(x, w, s, lhs_indices=lhs, rhs_indices=one, **KW), x, v, lhs, one)
    srt = torch.sort(rhs).values
    out = mq.gather_qmm(x, w, s, lhs_indices=lhs, rhs_indices=srt, sorted_indices=True, **KW)
    _check_gather(out, x, v, lhs, srt)


@pytest.mark.parametrize("P", [257, 1027, 16383, 16385, 32766, 32769, 70001])
@pytest.mark.parametrize("E", [3, 700])
def test_gather_sorts_any_number_of_pairs(P, E):
    g = _gen(P + E)
    N, K, B = 20, 64, 37
    w, s, v = weights(g, E, N, K)
    x = _randn(g, B, 1, K, dtype=torch.float16)
    # most pairs on one expert, many experts without any, some out of range
    rhs = (torch.rand(P, generator=g, device="cuda") ** 4 * (E + 1)).int()
    rhs[torch.randint(0, P, (P // 9,), generator=g, device="cuda")] = -3
    lhs = torch.randint(0, B, (P,), generator=g, device="cuda").int()
    lhs[P - 1], lhs[P // 2] = B, -1
    out = mq.gather_qmm(x, w, s, lhs_indices=lhs, rhs_indices=rhs, **KW)
    _check_gather(out, x, v, lhs, rhs)
    rhs[P - 3:] = E - 1                                      # the last pairs, no lhs
    out = mq.gather_qmm(x[:1], w, s, rhs_indices=rhs[1:], **KW)   # and 4-byte alignment
    _check_gather(out, x[:1], v, torch.zeros_like(rhs[1:]), rhs[1:])


@pytest.mark.parametrize("T,k,E,N,K", [(1500, 8, 400, 512, 2048), (300, 8, 100, 768, 1024),
                                       (2000, 4, 300, 260, 544)])
def test_gather_of_many_short_segments(T, k, E, N, K):
    """Tiles of few rows all over the chip, loads late under the traffic."""
    g = _gen(T + K)
    w, s, _ = weights(g, E * N, K)
    x = _randn(g, T, 1, 1, K, dtype=torch.bfloat16)
    p = torch.arange(1, E + 1, device="cuda").float() ** -1.0
    idx = torch.multinomial(p[torch.randperm(E, generator=g, device="cuda")].expand(T, E), k,
                            generator=g).int()
    bank = (w.reshape(E, N, -1), s.reshape(E, N, -1))
    for _ in range(3):
        out = mq.gather_qmm(x, *bank, rhs_indices=idx, **KW).reshape(T * k, N)
        flat = idx.reshape(-1)
        for e in range(0, E, 7):
            rows = (flat == e).nonzero().flatten()
            v = mq.dequantize(bank[0][e], bank[1][e], dtype=torch.float32, **KW).double()
            _check(out[rows], x.reshape(T, K)[rows // k], v, torch.bfloat16)


def test_gather_many_experts_in_slices():
    g = _gen(8)
    E, N, K, P = 2050, 16, 32, 400
    w, s, v = weights(g, E, N, K)
    x = _randn(g, P, 1, K, dtype=torch.bfloat16)
    rhs = torch.randint(0, E, (P,), generator=g, device="cuda")
    out = mq.gather_qmm(x, w, s, rhs_indices=rhs, **KW)
    _check_gather(out, x, v, torch.arange(P, device="cuda"), rhs)
    few = mq.gather_qmm(x[:9], w, s, rhs_indices=rhs[:9], **KW)
    _check_gather(few, x[:9], v, torch.arange(9, device="cuda"), rhs[:9])


def test_gather_composed_forms():
    g = _gen(9)
    w, s, v = weights(g, 3, 64, 96)
    rhs = torch.tensor([2, 0, 2, 5], device="cuda")
    xf = _randn(g, 4, 2, 96)
    out = mq.gather_qmm(xf, w, s, rhs_indices=rhs, **KW)
    assert out.dtype == torch.float32 and not out[3].any()
    y = torch.matmul(xf[:3].double(), v[rhs[:3]].transpose(1, 2).contiguous())
    assert torch.allclose(out[:3].double(), y, rtol=0, atol=1e-4)
    xt = _randn(g, 4, 1, 64, dtype=torch.bfloat16)            # w as [K=64, N=96]
    out = mq.gather_qmm(xt, w, s, rhs_indices=rhs, transpose=False, **KW)
    _check(out[0], xt[0], v[2].T.contiguous(), torch.bfloat16)


def test_products_of_rows_too_long_for_the_kernels():
    g = _gen(20)
    E, N, K = 2, 8, 32 * 9216
    w, s, v = weights(g, E, N, K)
    x = _randn(g, 3, 1, K, dtype=torch.bfloat16)
    rhs = torch.tensor([1, 0, 1], device="cuda")
    _check_gather(mq.gather_qmm(x, w, s, rhs_indices=rhs, **KW), x, v,
                  torch.arange(3, device="cuda"), rhs)
    _check(mq.quantized_matmul(x[:, 0], w[0], s[0], **KW), x[:, 0], v[0], torch.bfloat16)


def test_offsets_past_32_bits():
    g = _gen(10)
    # a bank whose last experts' codes lie past 4 GB
    E, N, K = 530, 2048, 8192
    w = torch.zeros(E, N, K // 8, dtype=torch.int32, device="cuda")
    s = torch.full((E, N, K // 32), 127, dtype=torch.uint8, device="cuda")
    w1, s1, v1 = weights(g, 64, K)
    w[E - 1, N - 64:] = w1.view(torch.int32)
    s[E - 1, N - 64:] = s1
    x = _randn(g, 3, 1, K, dtype=torch.bfloat16)
    out = mq.gather_qmm(x, w.view(torch.uint32), s,
                        rhs_indices=torch.tensor([E - 1, 0, E - 1], device="cuda"), **KW)
    assert not out[1].any() and not out[0, :, :N - 64].any()
    _check(out[0, :, N - 64:], x[0], v1, torch.bfloat16)
    _check(out[2, :, N - 64:], x[2], v1, torch.bfloat16)
    full = mq.quantized_matmul(x[:, 0], w.view(torch.uint32).reshape(E * N, -1),
                               s.reshape(E * N, -1), **KW)
    _check(full[:, -64:], x[:, 0], v1, torch.bfloat16)
    del w, s, full
    # x rows past 4 GB
    rows = (1 << 32) // (2 * K) + 7
    big = torch.zeros(rows, 1, K, dtype=torch.bfloat16, device="cuda")
    big[-1, 0] = x[0, 0]
    bank = (w1.reshape(1, 64, -1), s1.reshape(1, 64, -1))
    for P in (3, 400):
        lhs = torch.zeros(P, dtype=torch.int64, device="cuda")
        lhs[P - 1] = rows - 1
        out = mq.gather_qmm(big, *bank, lhs_indices=lhs, rhs_indices=torch.zeros_like(lhs), **KW)
        assert not out[:P - 1].any()
        _check(out[P - 1], x[0], v1, torch.bfloat16)
    tall = mq.quantized_matmul(big[:, 0], w1, s1, **KW)
    assert not tall[:-1].any()
    _check(tall[-1:], x[0], v1, torch.bfloat16)


# ---- streams, graphs, modules ----------------------------------------------------

def _calls(g):
    w, s, _ = weights(g, 200, 320)
    bw, bs, _ = weights(g, 12, 96, 320)
    x = _randn(g, 400, 320, dtype=torch.bfloat16)
    idx = torch.randint(0, 12, (400, 3), generator=g, device="cuda", dtype=torch.int32)

    def run():
        xq = mq.dequantize(*mq.quantize(x, **KW), **KW)
        return [xq, mq.quantized_matmul(x[:3], w, s, **KW), mq.quantized_matmul(x, w, s, **KW),
                mq.qqmm(x[:9], w, s), mq.qqmm(x, w, s),
                mq.gather_qmm(x[:2, None, None], bw, bs, rhs_indices=idx[:2], **KW),
                mq.gather_qmm(x[:, None, None], bw, bs, rhs_indices=idx, **KW)]
    return x, run


def test_side_stream():
    _, run = _calls(_gen(11))
    want = run()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = run()
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_graph_replays():
    x, run = _calls(_gen(12))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        run()
    torch.cuda.current_stream().wait_stream(st)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            out = run()
        graphs.append((graph, out))
    g = _gen(13)
    for i in range(4):
        x.copy_(_randn(g, 400, 320))
        want = run()                                          # eager work between the replays
        torch.cuda.synchronize()
        for graph, out in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_graphs_of_one_stream_replay_side_by_side():
    """Two graphs captured on one stream do not share a workspace."""
    st = torch.cuda.Stream()
    calls = [_calls(_gen(16)), _calls(_gen(17))]
    want = [run() for _, run in calls]
    graphs = []
    st.wait_stream(torch.cuda.current_stream())
    for _, run in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            out = run()
        graphs.append((graph, out))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(5):
        for s, (graph, out) in zip(streams, graphs):
            with torch.cuda.stream(s):
                for o in out:
                    o.zero_()
                graph.replay()
        torch.cuda.synchronize()
        for w, (_, out) in zip(want, graphs):
            assert all(torch.equal(a, b) for a, b in zip(out, w)), i


def test_threads_share_a_stream():
    calls = [_calls(_gen(18)), _calls(_gen(19))]
    want = [run() for _, run in calls]
    torch.cuda.synchronize()
    bad = []

    def work(k):
        for _ in range(40):
            got = calls[k][1]()
            bad.extend(k for a, b in zip(got, want[k]) if not torch.equal(a, b))

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not bad


def test_launches_are_counted():
    x, run = _calls(_gen(14))
    before = mq.launch_count()
    run()
    assert mq.launch_count() - before >= 8


def test_layers():
    g = _gen(15)
    wf = _randn(g, 150, 256, dtype=torch.bfloat16) * 0.02
    bias = _randn(g, 150, dtype=torch.bfloat16)
    lin = nn.QuantizedLinear.from_linear(wf, bias=bias, **KW)
    v = values_ref(*quantize_ref(wf))
    assert torch.equal(lin.dequantized_weight().double(), v)
    x = _randn(g, 2, 6, 256, dtype=torch.bfloat16)
    y = mq.quantized_matmul(x, lin.weight, lin.scales, **KW)
    _check(y.reshape(12, 150), x.reshape(12, 256), v, torch.bfloat16)
    assert torch.equal(lin(x), y + bias)
    qq = nn.QQLinear.from_linear(wf, bias=bias)
    assert torch.equal(qq(x), mq.qqmm(x, qq.weight, qq.scales) + bias)
    # to and from the affine format, in place
    model = torch.nn.ModuleDict({"lm_head": torch.nn.Linear(256, 150, device="cuda",
                                                            dtype=torch.bfloat16)})
    rebit.apply(model, "head=mxfp4")
    assert model["lm_head"].mode == "mxfp4"
    assert rebit.apply(model, "head=mxfp4") == {"head": 0}
    mxw = model["lm_head"].dequantized_weight()
    rebit.apply(model, "head=8:32")
    assert model["lm_head"].mode == "affine"
    near = (model["lm_head"].dequantized_weight() - mxw).abs().max()
    assert float(near) <= float(mxw.abs().max()) / 50


@pytest.mark.parametrize("T", [1, 5, 30, 400])
@pytest.mark.parametrize("fuse", [False, True])
def test_switch_glu(T, fuse):
    """Router's choice -> gate, up, down over MXFP4 banks, step by step in 64
    bits on the operators' own rounded intermediates."""
    g = _gen(T)
    E, k, H, I = 10, 4, 192, 96
    banks = [weights(g, E, I, H), weights(g, E, I, H), weights(g, E, H, I)]
    moe = nn.SwitchGLU(*[nn.QuantizedSwitchLinear(w, s, None, **KW) for w, s, _ in banks],
                       fuse_gate_up=fuse)
    x = _randn(g, T, H, dtype=torch.bfloat16) * 4
    logits = _randn(g, T, E)
    idx, wts = mq.moe_route(logits, k)[:2]
    out = moe(x, idx, wts)
    assert out.shape == (T, H)
    xe = x.reshape(T, 1, 1, H)
    gate = mq.gather_qmm(xe, *banks[0][:2], rhs_indices=idx, **KW)
    up = mq.gather_qmm(xe, *banks[1][:2], rhs_indices=idx, **KW)
    lhs = torch.arange(T, device="cuda").repeat_interleave(k)
    _check_gather(gate, x.reshape(T, 1, H), banks[0][2], lhs, idx.reshape(-1))
    h = ops.swiglu(gate, up)
    y = mq.gather_qmm(h, *banks[2][:2], rhs_indices=idx, **KW)
    _check_gather(y, h.reshape(T * k, 1, I), banks[2][2], torch.arange(T * k, device="cuda"),
                  idx.reshape(-1))
    assert torch.equal(out, mq.moe_combine(y.reshape(-1, H), None, wts, T, k))
    assert torch.equal(moe(x, idx), y.reshape(T, k, H))
    glu = ops.gather_glu(xe, *banks[0][:2], None, *banks[1][:2], None, rhs_indices=idx, **KW)
    want = torch.nn.functional.silu(gate.float()) * up.float()
    assert torch.equal(glu, want.to(glu.dtype))


@pytest.mark.parametrize("T", [1, 5, 400])
@pytest.mark.parametrize("fuse", [False, True])
@pytest.mark.parametrize("which", ["down", "gate and up", "up"])
def test_switch_glu_of_both_formats(T, fuse, which):
    g = _gen(T + 30)
    E, k, H, I = 10, 4, 192, 128
    wf = [_randn(g, E, *s, dtype=torch.bfloat16) * 0.05 for s in ((I, H), (I, H), (H, I))]
    mx = {"down": (2,), "gate and up": (0, 1), "up": (1,)}[which]
    proj = []
    for i, w in enumerate(wf):
        kw = KW if i in mx else dict(group_size=64, bits=4)
        q = mq.quantize(w, **kw)
        proj.append(nn.QuantizedSwitchLinear(q[0], q[1], None if i in mx else q[2], **kw))
    x = _randn(g, T, H, dtype=torch.bfloat16)
    idx, wts = mq.moe_route(_randn(g, T, E), k)[:2]
    out = nn.SwitchGLU(*proj, fuse_gate_up=fuse)(x, idx, wts)
    xe = x[:, None, None]
    if fuse and T < 400 and which == "down":
        a, b = proj[:2]
        h = ops.gather_glu(xe, a.weight, a.scales, a.biases, b.weight, b.scales, b.biases,
                           rhs_indices=idx, group_size=64, bits=4)
    else:
        h = ops.swiglu(proj[0](xe, idx), proj[1](xe, idx))
    y = proj[2](h, idx)
    assert torch.equal(out, mq.moe_combine(y.reshape(-1, H), None, wts, T, k))
