"""quantized_glu and the gradients past quantized weights against 64-bit references
(glu_helpers.py): every kernel, at the sizes, strides and values where they can go
wrong."""

import pytest
import torch

import mlxturbo_amd as mq
from glu_helpers import ACTS, bank, check, glu_grad_ref, glu_ref, matmul_ref

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def _gen(seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _case(M, N, K, gs, bits, dtype, seed=0):
    g = _gen(seed)
    gate, wg = bank(g, N, K, gs, bits, dtype)
    up, wu = bank(g, N, K, gs, bits, dtype)
    x = torch.randn((M, K), generator=g, device="cuda").to(dtype)
    return g, x, gate, wg, up, wu


# rows of every kernel and its edges; columns ragged against tiles of 8, 128 and 256;
# K of one group, of odd numbers of groups, of whole units and of several slices
SHAPES = [
    (1, 1, 32, 32, 4, BF, "silu"),
    (1, 130, 64, 64, 8, HF, "gelu_tanh"),
    (1, 4099, 512, 64, 4, BF, "silu"),
    (2, 257, 96, 32, 4, HF, "silu"),
    (3, 64, 320, 64, 4, BF, "gelu_tanh"),
    (5, 1001, 1024, 32, 4, BF, "silu"),
    (8, 2056, 2048, 128, 4, HF, "silu"),
    (8, 520, 20480, 64, 4, BF, "silu"),
    (9, 72, 1280, 128, 8, BF, "gelu_tanh"),
    (13, 40, 640, 64, 8, HF, "silu"),
    (16, 300, 8192, 64, 8, BF, "silu"),
    (16, 35000, 256, 64, 4, BF, "silu"),
    (17, 129, 64, 64, 4, BF, "silu"),
    (20, 96, 96, 32, 8, BF, "silu"),
    (33, 1000, 192, 32, 4, HF, "gelu_tanh"),
    (64, 512, 1024, 64, 4, BF, "silu"),
    (100, 333, 640, 128, 8, HF, "silu"),
    (129, 640, 2560, 64, 8, BF, "gelu_tanh"),
    (300, 1111, 512, 32, 4, BF, "silu"),
    (1000, 2048, 1536, 64, 4, HF, "silu"),
]


@pytest.mark.parametrize("M,N,K,gs,bits,dtype,act", SHAPES)
def test_forward(M, N, K, gs, bits, dtype, act):
    _, x, gate, wg, up, wu = _case(M, N, K, gs, bits, dtype)
    before = mq.launch_count()
    h = mq.quantized_glu(x, gate, up, act, group_size=gs, bits=bits)
    assert mq.launch_count() > before and h.dtype == dtype and h.shape == (M, N)
    check(h, *glu_ref(x, wg, wu, act, dtype))


@pytest.mark.parametrize("M,N,K,gs,bits,dtype,act", SHAPES)
def test_gradient(M, N, K, gs, bits, dtype, act):
    g, x, gate, wg, up, wu = _case(M, N, K, gs, bits, dtype, seed=1)
    d = torch.randn((M, N), generator=g, device="cuda").to(dtype)
    x.requires_grad_()
    h = mq.quantized_glu(x, gate, up, act, group_size=gs, bits=bits)
    check(h.detach(), *glu_ref(x.detach(), wg, wu, act, dtype), "h")
    dx, = torch.autograd.grad(h, x, d)
    assert dx.dtype == dtype and dx.shape == x.shape
    check(dx, *glu_grad_ref(x.detach(), d, wg, wu, act, dtype), "dx")


@pytest.mark.parametrize("M,N,K,gs,bits,dtype", [s[:6] for s in SHAPES])
def test_matmul_gradient(M, N, K, gs, bits, dtype):
    g = _gen(2)
    b, w = bank(g, N, K, gs, bits, dtype)
    x = torch.randn((M, K), generator=g, device="cuda").to(dtype).requires_grad_()
    d = torch.randn((M, N), generator=g, device="cuda").to(dtype)
    y = mq.quantized_matmul(x, *b, group_size=gs, bits=bits)
    same = mq.quantized_matmul(x.detach(), *b, group_size=gs, bits=bits)
    assert torch.equal(y.detach(), same)
    dx, = torch.autograd.grad(y, x, d)
    check(dx, *matmul_ref(d, w.T, dtype), "dx")


@pytest.mark.parametrize("M", [1, 4, 40, 200])
@pytest.mark.parametrize("gs,bits,dtype", [(64, 4, BF), (32, 8, HF)])
def test_strides_and_alignment(M, gs, bits, dtype):
    """Leading dimensions, rows inside a longer buffer, transposed x, weights, scales and
    x at odd addresses."""
    K, N = 256, 130
    g, x, gate, wg, up, wu = _case(M, N, K, gs, bits, dtype, seed=3)
    kw = dict(group_size=gs, bits=bits)
    want = mq.quantized_glu(x, gate, up, **kw)
    wide = torch.randn((M, 2 * K + 3), generator=g, device="cuda").to(dtype)
    wide[:, 1:K + 1] = x
    for v in (x.reshape(1, M, 1, K), wide[:, 1:K + 1], x.t().contiguous().t()):
        got = mq.quantized_glu(v, gate, up, **kw)
        assert got.shape == (*v.shape[:-1], N) and torch.equal(got.reshape(M, N), want)

    def odd(t):
        """The same values two bytes (words: four) past an aligned address."""
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        buf[1:] = t.reshape(-1)
        return buf[1:].view(t.shape)

    got = mq.quantized_glu(odd(x), tuple(map(odd, gate)), tuple(map(odd, up)), **kw)
    assert torch.equal(got, want)
    xg = wide[:, 1:K + 1].requires_grad_()
    d = torch.randn((M, N), generator=g, device="cuda").to(dtype)
    dx, = torch.autograd.grad(mq.quantized_glu(xg, gate, up, **kw), xg, odd(d))
    check(dx, *glu_grad_ref(x, d, wg, wu, "silu", dtype))
    # a gradient that is one number everywhere
    dx, = torch.autograd.grad(mq.quantized_glu(xg, gate, up, **kw).sum(), xg)
    check(dx, *glu_grad_ref(x, torch.ones((M, N), device="cuda").to(dtype), wg, wu, "silu", dtype))


def test_scales_at_two_byte_addresses():
    """The C entry with scales and biases between dwords (the operators copy those)."""
    from mlxturbo_amd import _lib
    N, K = 40, 512
    for M in (3, 30):
        _, x, gate, wg, up, wu = _case(M, N, K, 64, 4, BF, seed=4)
        flat = []
        for w, s, b in (gate, up):
            flat.append(w)
            for t in (s, b):
                buf = torch.empty(t.numel() + 1, dtype=BF, device="cuda")
                buf[1:] = t.reshape(-1)
                flat.append(buf[1:])
        out = torch.empty((M, N), dtype=BF, device="cuda")
        rc = _lib.lib().mq_quantized_glu(x.data_ptr(), *[t.data_ptr() for t in flat],
                                         out.data_ptr(), None, None, M, N, K, 64, 4, 0, 0, None,
                                         0, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        check(out, *glu_ref(x, wg, wu, "silu", BF))


@pytest.mark.parametrize("M", [1, 7, 40, 300])
@pytest.mark.parametrize("bits", [4, 8])
def test_large_scales(M, bits):
    """Scales of 2^100 and more take the float route of every kernel, forward and back:
    the sums overflow or not as the definition's."""
    N, K, gs = 70, 512, 64
    g, x, gate, wg, up, wu = _case(M, N, K, gs, bits, BF, seed=5)
    x = (x.float() * 2.0 ** -100).to(BF)
    for m, w in ((gate, wg), (up, wu)):
        for n in (0, 13, 69):
            m[1][n, 3] = 2.0 ** 101
    from glu_helpers import values
    code = [_codes(m[0], bits) for m in (gate, up)]
    wg, wu = (values(c, m[1], m[2], gs) for c, m in zip(code, (gate, up)))
    xg = x.clone().requires_grad_()
    h = mq.quantized_glu(xg, gate, up, group_size=gs, bits=bits)
    check(h.detach(), *glu_ref(x, wg, wu, "silu", BF), "h")
    d = (torch.randn((M, N), generator=g, device="cuda") * 2.0 ** -60).to(BF)
    dx, = torch.autograd.grad(h, xg, d)
    check(dx, *glu_grad_ref(x, d, wg, wu, "silu", BF), "dx")


def _codes(w, bits):
    b = w.view(torch.int32).view(torch.uint8).long()
    if bits == 8:
        return b
    return torch.stack([b & 15, b >> 4], -1).reshape(b.shape[0], -1)


@pytest.mark.parametrize("M", [5, 16, 90])
def test_rows_do_not_meet(M):
    """A row of NaN, infinities or nothing changes its own results alone."""
    N, K = 200, 1024
    g, x, gate, _, up, _ = _case(M, N, K, 64, 4, BF, seed=6)
    d = torch.randn((M, N), generator=g, device="cuda").to(BF)

    def both(x, d):
        xg = x.clone().requires_grad_()
        h = mq.quantized_glu(xg, gate, up)
        return h.detach(), torch.autograd.grad(h, xg, d)[0]

    h0, dx0 = both(x, d)
    x1, d1 = x.clone(), d.clone()
    x1[1], x1[3, 5] = float("nan"), float("inf")
    d1[2] = float("nan")
    h1, dx1 = both(x1, d1)
    rest = [r for r in range(M) if r not in (1, 3)]
    assert torch.equal(h1[rest], h0[rest])
    rest = [r for r in rest if r != 2]
    assert torch.equal(dx1[rest], dx0[rest])
    assert h1[1].isnan().all() and dx1[2].isnan().all()


def test_matmul_gradient_ragged_rows_of_nan():
    """N that is not whole steps: the next row's values are not read into a row's sum."""
    g = _gen(7)
    b, w = bank(g, 100, 256, 64, 4, BF)
    x = torch.randn((6, 256), generator=g, device="cuda").to(BF).requires_grad_()
    d = torch.randn((6, 100), generator=g, device="cuda").to(BF)
    d[3] = float("nan")
    dx, = torch.autograd.grad(mq.quantized_matmul(x, *b), x, d)
    rest = [0, 1, 2, 4, 5]
    check(dx[rest], *(t[rest] for t in matmul_ref(d.nan_to_num(0), w.T, BF)))
    assert dx[3].isnan().all()


@pytest.mark.parametrize("lead", [(0,), (2, 0), ()])
def test_empty_and_scalar_leads(lead):
    _, _, gate, _, up, _ = _case(1, 24, 64, 64, 4, BF)
    x = torch.ones((*lead, 64), dtype=BF, device="cuda", requires_grad=True)
    h = mq.quantized_glu(x, gate, up)
    assert h.shape == (*lead, 24)
    h.sum().backward()
    assert x.grad.shape == x.shape
    none = tuple(t[:0] for t in gate)
    h = mq.quantized_glu(x, none, none)
    assert h.shape == (*lead, 0)
    x.grad = None
    h.sum().backward()
    assert not x.grad.any()


@pytest.mark.parametrize("kw", [dict(bits=3), dict(bits=6, dtype=HF), dict(x=torch.float32)], ids=str)
def test_composed_formats(kw):
    """Formats without kernels: two products, rounded, and the activation; x's gradient as
    torch makes it of the composed product."""
    dtype, bits = kw.get("dtype", BF), kw.get("bits", 4)
    xt = kw.get("x", dtype)
    g = _gen(8)
    w = [(torch.randn((48, 128), generator=g, device="cuda") * 0.05).to(dtype) for _ in range(2)]
    banks = [mq.quantize(v, 64, bits) for v in w]
    x = torch.randn((5, 128), generator=g, device="cuda").to(xt).requires_grad_()
    h = mq.quantized_glu(x, *banks, group_size=64, bits=bits)
    gv, uv = (mq.quantized_matmul(x, *b, group_size=64, bits=bits) for b in banks)
    want = (torch.nn.functional.silu(gv.float()) * uv.float()).to(gv.dtype)
    assert h.dtype == want.dtype and torch.equal(h, want)
    d = torch.randn(h.shape, generator=g, device="cuda").to(h.dtype)
    assert torch.equal(torch.autograd.grad(h, x, d)[0], torch.autograd.grad(want, x, d)[0])


def test_mxfp4():
    g = _gen(9)
    banks = [mq.quantize(torch.randn((64, 128), generator=g, device="cuda").to(BF), mode="mxfp4")
             for _ in range(2)]
    x = torch.randn((5, 128), generator=g, device="cuda").to(BF)
    h = mq.quantized_glu(x, *banks, activation="gelu_tanh", mode="mxfp4")
    gv, uv = (mq.quantized_matmul(x, *b, mode="mxfp4") for b in banks)
    want = torch.nn.functional.gelu(gv.float(), approximate="tanh") * uv.float()
    assert torch.equal(h, want.to(BF))
    with pytest.raises(NotImplementedError, match="gradients"):
        mq.quantized_glu(x.requires_grad_(), *banks, mode="mxfp4")


def test_refusals():
    _, x, gate, _, up, _ = _case(2, 24, 128, 64, 4, BF)
    with pytest.raises(ValueError, match="does not match"):
        mq.quantized_glu(x[:, :64], gate, up)
    with pytest.raises(ValueError, match="differ"):
        mq.quantized_glu(x, gate, tuple(t[:-1] for t in up))
    with pytest.raises(ValueError, match="differ"):
        mq.quantized_glu(x, gate, (up[0], up[1].half(), up[2].half()))
    with pytest.raises(ValueError, match="biases"):
        mq.quantized_glu(x, (*gate[:2], None), up)
    with pytest.raises(NotImplementedError, match="2-D"):
        mq.quantized_glu(x, tuple(t[None] for t in gate), tuple(t[None] for t in up))
    with pytest.raises(NotImplementedError, match="only affine"):
        mq.quantized_glu(x, gate, up, mode="nvfp4")
    x.requires_grad_()
    s = gate[1].clone().requires_grad_()
    with pytest.raises(NotImplementedError, match="constants"):
        mq.quantized_glu(x, (gate[0], s, gate[2]), up)
    with pytest.raises(NotImplementedError, match="constants"):
        mq.quantized_matmul(x, gate[0], s, gate[2])
    # a second derivative
    h = mq.quantized_glu(x, gate, up)
    dx, = torch.autograd.grad(h.float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
    # weights changed between forward and backward
    h = mq.quantized_glu(x, gate, up)
    gate[1].mul_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        h.sum().backward()


def test_no_grad_is_the_plain_call():
    _, x, gate, _, up, _ = _case(20, 240, 128, 64, 4, BF)
    want = mq.quantized_glu(x, gate, up)
    x.requires_grad_()
    with torch.no_grad():
        h = mq.quantized_glu(x, gate, up)
        y = mq.quantized_matmul(x, *gate)
    assert not h.requires_grad and not y.requires_grad and torch.equal(h, want)
    # the sums kept for the gradient leave the result as it is
    assert torch.equal(mq.quantized_glu(x, gate, up).detach(), want)


def _mlp(g, H, I, dtype, bits=4, **kw):
    from mlxturbo_amd.nn import QuantizedLinear, QuantizedMLP

    def layer(n, k):
        w = (torch.randn((n, k), generator=g, device="cuda") * k ** -0.5).to(dtype)
        return QuantizedLinear.from_linear(w, bits=bits)
    return QuantizedMLP(layer(I, H), layer(I, H), layer(H, I), **kw)


@pytest.mark.parametrize("rows", [1, 6, 130])
@pytest.mark.parametrize("act", ACTS)
def test_mlp_is_its_steps(rows, act):
    """The module's forward and its gradient are the three operators' in turn."""
    g = _gen(10)
    mlp = _mlp(g, 256, 704, BF, activation=act)
    x = torch.randn((2, rows, 256), generator=g, device="cuda").to(BF).requires_grad_()
    y = mlp(x)
    banks = [(m.weight, m.scales, m.biases) for m in (mlp.gate_proj, mlp.up_proj, mlp.down_proj)]
    h = mq.quantized_glu(x, banks[0], banks[1], act)
    want = mq.quantized_matmul(h, *banks[2])
    assert torch.equal(y, want)
    d = torch.randn(y.shape, generator=g, device="cuda").to(BF)
    dx, = torch.autograd.grad(y, x, d)
    dh, = torch.autograd.grad(want, h, d, retain_graph=True)
    wg, wu, wd = (mq.dequantize(*b).double() for b in banks)
    check(dh.reshape(-1, 704), *matmul_ref(d.reshape(-1, 256), wd.T, BF))
    check(dx.reshape(-1, 256), *glu_grad_ref(x.detach().reshape(-1, 256), dh.reshape(-1, 704), wg,
                                             wu, act, BF))


def test_mlp_with_biases_and_formats():
    from mlxturbo_amd.nn import QuantizedLinear, QuantizedMLP
    g = _gen(11)
    w = [(torch.randn((n, k), generator=g, device="cuda") * 0.05).to(BF)
         for n, k in ((96, 128), (96, 128), (128, 96))]
    x = torch.randn((3, 128), generator=g, device="cuda").to(BF)
    bias = torch.randn(96, generator=g, device="cuda").to(BF)
    for gate in (QuantizedLinear.from_linear(w[0], bias=bias, group_size=32),
                 QuantizedLinear.from_linear(w[0], bits=8, group_size=32),
                 QuantizedLinear.from_linear(w[0], mode="mxfp4")):
        mlp = QuantizedMLP(gate, QuantizedLinear.from_linear(w[1], group_size=32),
                           QuantizedLinear.from_linear(w[2], group_size=32))
        h = torch.nn.functional.silu(mlp.gate_proj(x).float()) * mlp.up_proj(x).float()
        assert torch.equal(mlp(x), mlp.down_proj(h.to(BF)))
    with pytest.raises(ValueError, match="activation"):
        QuantizedMLP(gate, gate, gate, activation="relu")


def test_graph_of_a_step():
    """A training step captured with a leaf of its own, replayed between eager work."""
    g = _gen(12)
    mlp = _mlp(g, 256, 704, BF)
    x = torch.randn((130, 256), generator=g, device="cuda").to(BF)
    d = torch.randn((130, 256), generator=g, device="cuda").to(BF)

    def step():
        leaf = x.detach().requires_grad_()
        y = mlp(leaf)
        return y.detach(), torch.autograd.grad(y, leaf, d)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dx = step()
    for i in range(4):
        x.copy_(torch.randn(x.shape, generator=g, device="cuda").to(BF))
        d.copy_(torch.randn(d.shape, generator=g, device="cuda").to(BF))
        eager = mq.quantized_matmul(x, mlp.gate_proj.weight, mlp.gate_proj.scales,
                                    mlp.gate_proj.biases)
        graph.replay()
        torch.cuda.synchronize()
        assert eager.shape == (130, 704)
        want = step()
        assert torch.equal(y, want[0]) and torch.equal(dx, want[1])


def test_leaf_of_a_living_graph_is_refused_in_a_capture():
    g = _gen(13)
    mlp = _mlp(g, 128, 256, BF)
    x = torch.randn((4, 128), generator=g, device="cuda").to(BF).requires_grad_()
    alive = mlp(x)                                    # on the default stream
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="still lives"):
        with torch.cuda.graph(graph):
            mlp(x)
    torch.cuda.synchronize()
    alive.sum().backward()
    assert x.grad is not None
    del alive
    # without it, and with the graph's own leaf, the call can be captured
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = mlp(x.detach().requires_grad_())
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y.detach(), mlp(x).detach())


def test_streams_at_once():
    """Calls on two streams at once, K split in both, each with its own workspace."""
    g = _gen(14)
    cases = [_case(100, 256, 4096, 64, 4, BF, seed=20 + i)[1:] for i in range(2)]
    want = [mq.quantized_glu(x, gate, up) for x, gate, _, up, _ in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(8):
        for i, (x, gate, _, up, _) in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i].append(mq.quantized_glu(x, gate, up))
    torch.cuda.synchronize()
    assert all(torch.equal(h, want[i]) for i in range(2) for h in got[i])


# One row: waves of whole quads and of split ones (more quads than SIMDs, a leftover), K split
# over 2 and 4 waves, rows that end inside a load and their scales' last chunk, scales past
# the copy (then the kernel of 2 to 16 rows).  2 to 16 rows: scales of single entries and of
# eights, more of either than the threads read ahead; x in slices.  Split sums of odd
# widths.
MORE = [
    (1, 4099, 2048, 64, 4, BF, "silu"),
    (1, 2057, 2048, 128, 8, HF, "silu"),
    (1, 40, 20480, 32, 4, BF, "gelu_tanh"),
    (1, 131, 544, 32, 4, HF, "silu"),
    (1, 77, 800, 32, 8, BF, "silu"),
    (1, 24, 131072, 32, 4, BF, "silu"),
    (1, 3, 32, 32, 8, HF, "silu"),
    (2, 17000, 4096, 32, 4, BF, "silu"),
    (4, 17000, 960, 64, 4, BF, "silu"),
    (6, 9, 1056, 32, 8, HF, "silu"),
    (16, 2100, 10240, 128, 4, BF, "gelu_tanh"),
    (45, 1001, 2560, 128, 8, HF, "silu"),
    (64, 513, 4096, 64, 4, BF, "silu"),
]


@pytest.mark.parametrize("M,N,K,gs,bits,dtype,act", MORE)
def test_more_forward(M, N, K, gs, bits, dtype, act):
    _, x, gate, wg, up, wu = _case(M, N, K, gs, bits, dtype, seed=7)
    h = mq.quantized_glu(x, gate, up, act, group_size=gs, bits=bits)
    check(h, *glu_ref(x, wg, wu, act, dtype))
    # the sums kept for the gradient leave the result as it is
    x.requires_grad_()
    assert torch.equal(mq.quantized_glu(x, gate, up, act, group_size=gs, bits=bits).detach(), h)


@pytest.mark.parametrize("M,N,K,gs,bits,dtype,act", MORE)
def test_more_gradient(M, N, K, gs, bits, dtype, act):
    g, x, gate, wg, up, wu = _case(M, N, K, gs, bits, dtype, seed=8)
    d = torch.randn((M, N), generator=g, device="cuda").to(dtype)
    x.requires_grad_()
    h = mq.quantized_glu(x, gate, up, act, group_size=gs, bits=bits)
    dx, = torch.autograd.grad(h, x, d)
    check(dx, *glu_grad_ref(x.detach(), d, wg, wu, act, dtype), "dx")


@pytest.mark.parametrize("bits,dtype", [(4, BF), (8, HF)])
def test_one_row_scales_at_any_address(bits, dtype):
    """Scales and biases from two-byte addresses: every value of the same bits."""
    _, x, gate, _, up, _ = _case(1, 515, 1056, 32, bits, dtype, seed=9)
    kw = dict(group_size=32, bits=bits)
    want = mq.quantized_glu(x, gate, up, **kw)
    lib = mq._lib.lib()
    moved = []
    for m in (gate, up):
        moved.append(m[0])
        for t in m[1:]:
            buf = torch.full((t.numel() + 8,), float("nan"), dtype=dtype, device="cuda")
            buf[3:3 + t.numel()] = t.reshape(-1)
            moved.append(buf[3:3 + t.numel()])
    out = torch.full_like(want, float("nan"))
    rc = lib.mq_quantized_glu(x.data_ptr(), *[t.data_ptr() for t in moved], out.data_ptr(), None,
                              None, 1, 515, 1056, 32, bits, 0 if dtype == BF else 1, 0, None, 0,
                              torch.cuda.current_stream().cuda_stream)
    assert rc == 0 and torch.equal(out, want)


def test_weights_replaced_or_changed():
    """Like a saved tensor of the engine's: a weight changed in place since the forward pass
    is refused, and a graph can be gone through twice if it is kept."""
    _, x, gate, _, up, _ = _case(20, 240, 128, 64, 4, BF, seed=10)
    x.requires_grad_()
    h = mq.quantized_glu(x, gate, up)
    y = mq.quantized_matmul(x, *gate)
    first = [torch.autograd.grad(t.float().sum(), x, retain_graph=True)[0] for t in (h, y)]
    again = [torch.autograd.grad(t.float().sum(), x, retain_graph=True)[0] for t in (h, y)]
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    up[2].add_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        h.sum().backward(retain_graph=True)
    y.sum().backward(retain_graph=True)
    gate[0].copy_(gate[0].clone())
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


@pytest.mark.parametrize("shape", [(4, 128), (2, 2, 128)])
@pytest.mark.parametrize("glu", [False, True])
def test_every_call_notes_its_leaf(shape, glu):
    """The refusal above of either operator alone, of rows and of more dimensions, by a
    graph of the other one too."""
    _, x, gate, _, up, _ = _case(4, 256, 128, 64, 4, BF, seed=15)
    x = x.reshape(shape).requires_grad_()
    calls = [lambda t: mq.quantized_matmul(t, *gate), lambda t: mq.quantized_glu(t, gate, up)]
    for other in (False, True):
        alive = calls[glu](x)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="still lives"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                calls[other](x)
        torch.cuda.synchronize()
        del alive
