"""The gated block's gradient against its definition in 64 bits: that it is rounded once, and
that what lies between h's gradient and x's may be larger than the type holds."""

import pytest
import torch

import mlxturbo_amd as mq
from glu_helpers import activation, bank, check
from mlxturbo_amd import glu

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _case(M, N, K, gs, bits, dtype, seed, scale=0.02):
    g = _gen(seed)
    gate, wg = bank(g, N, K, gs, bits, dtype, scale=scale)
    up, wu = bank(g, N, K, gs, bits, dtype, scale=scale)
    x = torch.randn((M, K), generator=g, device="cuda").to(dtype)
    return g, x, gate, wg, up, wu


def _grad(x, gate, up, act, gs, bits, d):
    x = x.clone().requires_grad_()
    return torch.autograd.grad(mq.quantized_glu(x, gate, up, act, group_size=gs, bits=bits), x, d)[0]


def _between(x, d, wg, wu, act):
    """dL/dg and dL/du in float64, and how far the float ones may be: of the sums over K
    products, an addition 2^-23 of the sum of magnitudes (|act'| < 1.13, |act''| < 1.2), of the
    activation's float steps (16, and an exponent's error times |g|), and of the two products."""
    x, d = x.double(), d.double()
    g, u = x @ wg.T, x @ wu.T
    a, da = activation(g, act)
    eg, eu = ((x.shape[1] + 16) * 2.0 ** -23 * (x.abs() @ w.abs().T) for w in (wg, wu))
    rel = (18 + 4 * g.abs()) * 2.0 ** -23
    dg, du = d * u * da, d * a
    edg = d.abs() * ((u.abs() + eu) * (1.2 * eg + rel * 1.2) + eu * da.abs())
    edu = d.abs() * (1.13 * eg + rel * a.abs() + 2.0 ** -126)
    return dg, du, edg, edu


def _half_step(y, dtype):
    f = torch.finfo(dtype)
    return (f.eps / 2) * y.abs() + f.smallest_normal * f.eps / 2


def _pair(v, dtype):
    """What two numbers of a type leave of a value: half a step of half a step."""
    return (torch.finfo(dtype).eps / 2) ** 2 * v.abs() + _half_step(0 * v, dtype)


ONE_COLUMN = [
    (1, 40, 64, 64, 4, BF, "silu"),
    (7, 9, 64, 32, 8, HF, "gelu_tanh"),
    (33, 65, 96, 32, 4, BF, "gelu_tanh"),
    (64, 128, 128, 128, 4, HF, "silu"),
    (130, 300, 192, 64, 8, BF, "silu"),
    (300, 77, 128, 64, 4, HF, "gelu_tanh"),
]


@pytest.mark.parametrize("M,N,K,gs,bits,dtype,act", ONE_COLUMN)
def test_rounded_once(M, N, K, gs, bits, dtype, act):
    """h's gradient in one column of each row: x's is two products, whose error is the last
    rounding's and little else."""
    g, x, gate, wg, up, wu = _case(M, N, K, gs, bits, dtype, 1)
    d = torch.zeros((M, N), dtype=dtype, device="cuda")
    rows = torch.arange(M, device="cuda")
    d[rows, rows * 5 % N] = (1 + torch.rand(M, generator=g, device="cuda")).to(dtype)
    dg, du, edg, edu = _between(x, d, wg, wu, act)
    edg, edu = (e + _pair(v.abs() + e, dtype) for v, e in ((dg, edg), (du, edu)))
    edg, edu = edg * (d != 0), edu * (d != 0)
    # the sums: four products that are not 0, so a handful of roundings
    off = edg @ wg.abs() + edu @ wu.abs()
    off += 2.0 ** -20 * (dg.abs() @ wg.abs() + du.abs() @ wu.abs())
    dx = dg @ wg + du @ wu
    check(_grad(x, gate, up, act, gs, bits, d), dx, off + _half_step(dx.abs() + off, dtype))


ALL_COLUMNS = [
    (17, 1111, 512, 64, 4, BF, "silu"),
    (45, 1001, 2560, 128, 8, HF, "silu"),
    (129, 640, 1024, 64, 8, BF, "gelu_tanh"),
    (301, 2048, 1024, 32, 4, HF, "gelu_tanh"),
    (515, 2056, 640, 64, 4, BF, "silu"),
]


@pytest.mark.parametrize("M,N,K,gs,bits,dtype,act", ALL_COLUMNS)
def test_error_is_that_of_one_rounding(M, N, K, gs, bits, dtype, act):
    """Over all columns, the error's root mean square is that of rounding the exact gradient,
    to a tenth.  A number rounded to half a step eps / 2 is off by about eps / 5 in the mean
    square.  To it come, independent of it, the rests that pairs leave (eps^2 / 4 of each term at
    most) and the float sums' roundings: of about sqrt(4 N) additions 2^-23 each, 2^-16 of the
    result at N = 2056, where eps / 5 is 2^-9.3 (bfloat16) and 2^-12.3; so 1.01 at most.  One
    more rounding of the terms to the type makes it 1.41."""
    g, x, gate, wg, up, wu = _case(M, N, K, gs, bits, dtype, 2)
    d = torch.randn((M, N), generator=g, device="cuda").to(dtype)
    dg, du, _, _ = _between(x, d, wg, wu, act)
    dx = dg @ wg + du @ wu
    got = _grad(x, gate, up, act, gs, bits, d)
    err, least = (got.double() - dx).norm(), (dx.to(dtype).double() - dx).norm()
    assert float(err) < 1.1 * float(least), (float(err), float(least))
    # and the same bits again
    assert torch.equal(got, _grad(x, gate, up, act, gs, bits, d))


@pytest.mark.parametrize("dtype", [BF, HF])
def test_sizes_without_a_kernel(dtype, monkeypatch):
    """Sizes that the C entry refuses: float products over the dequantized weights."""
    g, x, gate, wg, up, wu = _case(5, 200, 128, 64, 4, dtype, 3)
    d = torch.randn((5, 200), generator=g, device="cuda").to(dtype)
    want = _grad(x, gate, up, "silu", 64, 4, d)
    lib = mq._lib.lib()

    class Refusing:
        def __getattr__(self, name):
            return getattr(lib, name)

        def mq_quantized_glu_grad(self, *args):
            return glu.ops._EUNSUPPORTED

    monkeypatch.setattr(glu._lib, "lib", Refusing)
    got = _grad(x, gate, up, "silu", 64, 4, d)
    dg, du, edg, edu = _between(x, d, wg, wu, "silu")
    dx = dg @ wg + du @ wu
    off = (edg + _pair(dg, dtype)) @ wg.abs() + (edu + _pair(du, dtype)) @ wu.abs()
    off += 450 * 2.0 ** -23 * (dg.abs() @ wg.abs() + du.abs() @ wu.abs())
    for v in (got, want):
        check(v, dx, off + _half_step(dx.abs() + off, dtype))


@pytest.mark.parametrize("M,bits", [(1, 4), (6, 8), (40, 4), (300, 4)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_range_between(M, bits, dtype):
    """A scaled loss' gradient and an activation far out: dL/dg and dL/du pass float16's
    range, and x's gradient does not.  Other rows are ordinary, tiny, or of zeros."""
    N, K = 200, 128
    g, x, gate, wg, up, wu = _case(M, N, K, 64, bits, dtype, 4)
    d = torch.randn((M, N), generator=g, device="cuda").to(dtype)
    x[0] = (x[0].float() * 400).to(dtype)
    gv, uv = (x[0].double() @ w.T for w in (wg, wu))
    av, dav = activation(gv, "silu")
    d[0] = 0
    d[0, (dav * uv).abs().argmax()], d[0, av.argmax()] = 600, -400
    if M > 4:
        d[1] = 0
        d[2] = (d[2].float() * 2.0 ** -12).to(dtype)
        x[3] = 0
    dg, du, edg, edu = _between(x, d, wg, wu, "silu")
    dx = dg @ wg + du @ wu
    assert float(dg.abs().max()) > 65504 and float(du.abs().max()) > 65504
    assert float(dx.abs().max()) < 60000
    got = _grad(x, gate, up, "silu", 64, bits, d)
    # a pair's last place: 2^-25 of float16 on rows whose largest is 2^14 at least
    last = 2.0 ** -39 * torch.maximum(dg.abs().amax(-1), du.abs().amax(-1))[:, None]
    rel = (torch.finfo(dtype).eps / 2) ** 2
    off = (edg + rel * dg.abs() + last) @ wg.abs() + (edu + rel * du.abs() + last) @ wu.abs()
    off += (2 * N + 20) * 2.0 ** -23 * (dg.abs() @ wg.abs() + du.abs() @ wu.abs())
    check(got, dx, off + _half_step(dx.abs() + off, dtype))
    if M > 4:
        assert not got[1].any()


def test_rows_with_infinities():
    """In float16 a row's factor is of its finite values, and rows that hold an infinity or
    a NaN stay apart from the others."""
    g, x, gate, wg, up, wu = _case(9, 72, 128, 64, 4, HF, 5)
    d = torch.randn((9, 72), generator=g, device="cuda").to(HF)
    want = _grad(x, gate, up, "silu", 64, 4, d)
    d[2, 5], d[4, 7], d[4, 8] = float("inf"), float("nan"), 3.0
    got = _grad(x, gate, up, "silu", 64, 4, d)
    rest = [r for r in range(9) if r not in (2, 4)]
    assert torch.equal(got[rest], want[rest])
    assert not got[2].isfinite().any() and got[4].isnan().all()


@pytest.mark.parametrize("both", [False, True])
@pytest.mark.parametrize("M,N,K", [(40, 1500, 256), (2100, 64, 8192)])
def test_gradient_at_any_address(M, N, K, both):
    """The C entries with x's gradient at two-byte addresses, its sums split and whole: the
    same bits, and nothing written beside them."""
    lib = mq._lib.lib()
    g, x, gate, _, up, _ = _case(M, N, K, 64, 4, BF, 6)
    d = torch.randn((M, N), generator=g, device="cuda").to(BF)
    sums = [torch.randn((M, N), generator=g, device="cuda") for _ in range(2)]
    size = lib.mq_quantized_glu_grad_workspace_size if both else lib.mq_quantized_matmul_grad_workspace_size
    ws = torch.empty(size(M, N, K, 64, 4), dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    got = []
    for off in (0, 1, 2, 4):
        buf = torch.full((M * K + 16,), 7.0, dtype=BF, device="cuda")
        dx = buf[off:].data_ptr()
        if both:
            rc = lib.mq_quantized_glu_grad(
                d.data_ptr(), *[t.data_ptr() for t in (*sums, *gate, *up)], dx, M, N, K, 64, 4, 0,
                0, ws.data_ptr(), ws.numel(), stream)
        else:
            rc = lib.mq_quantized_matmul_grad(
                d.data_ptr(), *[t.data_ptr() for t in gate], dx, M, N, K, 64, 4, 0, ws.data_ptr(),
                ws.numel(), stream)
        assert rc == 0
        assert (buf[:off] == 7).all() and (buf[off + M * K:] == 7).all()
        got.append(buf[off:off + M * K])
    assert got[0].isfinite().all() and all(torch.equal(t, got[0]) for t in got)


def test_streams_at_once_and_graphs():
    """float16 steps, whose rows' factors lie in the call's workspace: on two streams at once,
    and captured, both graphs replayed on streams of their own between eager steps."""
    cases = [_case(m, 512, 256, 64, 4, HF, 30 + m) for m in (40, 200)]
    ds = [torch.randn((x.shape[0], 512), generator=g, device="cuda").to(HF) for g, x, *_ in cases]

    def step(i):
        _, x, gate, _, up, _ = cases[i]
        leaf = x.detach().requires_grad_()
        return torch.autograd.grad(mq.quantized_glu(leaf, gate, up), leaf, ds[i])[0]

    want = [step(i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(i))
    torch.cuda.synchronize()
    assert all(torch.equal(v, want[i]) for i in range(2) for v in got[i])
    graphs, outs = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            outs.append(step(i))
    for n in range(4):
        for i in range(2):
            ds[i].mul_(-2.0 if n % 2 else 0.5)
        torch.cuda.synchronize()
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], step(i))
        torch.cuda.synchronize()
