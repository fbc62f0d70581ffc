"""x's gradient past MXFP4 weights, in the operator and in the layers that hold them."""

import pytest
import torch

import mlxturbo_amd as mq
from glu_helpers import check, matmul_ref
from mlxturbo_amd.nn import QQLinear, QuantizedLinear, QuantizedMLP

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _weight(g, n, k, dtype):
    return (torch.randn((n, k), generator=g, device="cuda") * k ** -0.5).to(dtype)


@pytest.mark.parametrize("lead,N,K,dtype", [((1,), 40, 64, BF), ((3, 5), 129, 96, HF),
                                            ((70,), 512, 256, BF), ((2, 1, 150), 77, 320, HF),
                                            ((), 8, 32, BF), ((0,), 24, 64, BF),
                                            ((4,), 96, 64, torch.float32)])
def test_matmul(lead, N, K, dtype):
    g = _gen(1)
    b = mq.quantize(_weight(g, N, K, dtype), mode="mxfp4")
    w = mq.dequantize(*b, mode="mxfp4", dtype=dtype).double()
    x = torch.randn((*lead, K), generator=g, device="cuda").to(dtype).requires_grad_()
    d = torch.randn((*lead, N), generator=g, device="cuda").to(dtype)
    y = mq.quantized_matmul(x, *b, mode="mxfp4")
    with torch.no_grad():
        assert torch.equal(y, mq.quantized_matmul(x, *b, mode="mxfp4"))
    dx, = torch.autograd.grad(y, x, d)
    assert dx.shape == x.shape and dx.dtype == dtype
    if x.numel():
        check(dx.reshape(-1, K), *matmul_ref(d.reshape(-1, N), w.T, dtype))


def test_matmul_against_differences():
    """d . (y(x + e) - y(x)) is dx . e: the products are linear, and each y is rounded."""
    g = _gen(2)
    b = mq.quantize(_weight(g, 200, 128, HF), mode="mxfp4")
    x = torch.randn((20, 128), generator=g, device="cuda").to(HF).requires_grad_()
    e = torch.randn((20, 128), generator=g, device="cuda").to(HF)
    x1 = (x + e).detach()
    e = x1.double() - x.detach().double()
    d = torch.randn((20, 200), generator=g, device="cuda").to(HF)
    y = mq.quantized_matmul(x, *b, mode="mxfp4")
    y1 = mq.quantized_matmul(x1, *b, mode="mxfp4")
    dx, = torch.autograd.grad(y, x, d)
    got = (d.double() * (y1.double() - y.detach().double())).sum()
    want = (dx.double() * e).sum()
    # half a step of each y and of each dx, and half as much again for the sums
    off = 1.5 * 2.0 ** -11 * ((d.double().abs() * (y1.double().abs() + y.detach().double().abs())).sum()
                              + (dx.double().abs() * e.abs()).sum())
    assert abs(float(got - want)) <= float(off)


def test_second_pass_and_changed_weights():
    g = _gen(3)
    b = mq.quantize(_weight(g, 64, 64, BF), mode="mxfp4")
    x = torch.randn((5, 64), generator=g, device="cuda").to(BF).requires_grad_()
    y = mq.quantized_matmul(x, *b, mode="mxfp4")
    dx, = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
    y = mq.quantized_matmul(x, *b, mode="mxfp4")
    b[1].add_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


@pytest.mark.parametrize("mx", ["g", "u", "d", "gu", "gd", "gud"])
def test_mlp(mx):
    """Gate, up and down in MXFP4 or affine: the gradient in a residual block is that of the
    layers one by one, each checked by itself here and in test_gpu_glu.py."""
    g = _gen(4)

    def layer(name, n, k):
        w = _weight(g, n, k, BF)
        if name in mx:
            return QuantizedLinear.from_linear(w, mode="mxfp4")
        return QuantizedLinear.from_linear(w, group_size=32)
    mlp = QuantizedMLP(layer("g", 96, 128), layer("u", 96, 128), layer("d", 128, 96))
    x = torch.randn((6, 128), generator=g, device="cuda").to(BF).requires_grad_()
    d = torch.randn((6, 128), generator=g, device="cuda").to(BF)
    dx, = torch.autograd.grad(x + mlp(x), x, d)
    # the steps in 64 bits
    wg, wu, wd = (m.dequantized_weight().double() for m in (mlp.gate_proj, mlp.up_proj,
                                                           mlp.down_proj))
    x64 = x.detach().double().requires_grad_()
    y64 = x64 + (torch.nn.functional.silu(x64 @ wg.T) * (x64 @ wu.T)) @ wd.T
    want, = torch.autograd.grad(y64, x64, d.double())
    # ten roundings of at most half a step, each of a term of the sums at most: of the products,
    # the activation's inputs, h, their gradients and the two parts of dx
    a = (x64 @ wg.T).detach()
    u = (x64 @ wu.T).detach()
    dh = d.double().abs() @ wd.abs()
    mag = (dh * u.abs() * 1.13) @ wg.abs() + (dh * (a.abs() + 0.3)) @ wu.abs() + d.double().abs()
    mag += (dh * 1.2 * a.abs() * u.abs()) @ wg.abs() + (dh * 1.13 * a.abs()) @ wu.abs()
    check(dx, want, 10 * 2.0 ** -8 * mag)
    assert float((dx.double() - want).norm() / want.norm()) < 10 * 2.0 ** -8


def test_qqmm_refuses_the_backward_pass():
    g = _gen(5)
    w = _weight(g, 64, 128, BF)
    lin = QQLinear.from_linear(w)
    x = torch.randn((5, 128), generator=g, device="cuda").to(BF)
    want = lin(x)
    x.requires_grad_()
    y = lin(x)
    assert torch.equal(y.detach(), want)
    with pytest.raises(NotImplementedError, match="qqmm"):
        (x + y[:, :1]).sum().backward()
    with torch.no_grad():
        assert not lin(x).requires_grad
    mlp = QuantizedMLP(lin, lin, QuantizedLinear.from_linear(w.t().contiguous(), mode="mxfp4"))
    with pytest.raises(NotImplementedError, match="qqmm"):
        mlp(x).sum().backward()


def test_graph_of_a_step():
    """A step through MXFP4 layers captured with a leaf of its own, replayed between eager
    work: every replay's gradient is the eager one."""
    g = _gen(6)
    mlp = QuantizedMLP(*(QuantizedLinear.from_linear(_weight(g, n, k, BF), mode="mxfp4")
                         for n, k in ((512, 256), (512, 256), (256, 512))))
    x = torch.randn((70, 256), generator=g, device="cuda").to(BF)
    d = torch.randn((70, 256), generator=g, device="cuda").to(BF)

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
    for _ in range(4):
        x.copy_(torch.randn(x.shape, generator=g, device="cuda").to(BF))
        d.copy_(torch.randn(d.shape, generator=g, device="cuda").to(BF))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and torch.equal(dx, want[1])
