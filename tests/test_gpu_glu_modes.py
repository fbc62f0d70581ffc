"""The gated block under the library's switches and in modules that are not plain."""

import pytest
import torch

import mlxturbo_amd as mq
from glu_helpers import bank
from mlxturbo_amd.nn import QuantizedLinear, QuantizedMLP

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


# K that the few-row kernel takes whole, and in slices for 16 rows but not for fewer;
# K that the many-row tile does not take
@pytest.mark.parametrize("N,K,gs,bits,dtype", [
    (2056, 2048, 64, 4, BF), (17408, 5120, 64, 4, BF), (300, 8192, 64, 8, HF), (520, 20480, 64, 4, BF),
    (72, 96, 32, 4, HF), (1001, 2560, 128, 8, BF), (264, 4128, 32, 8, BF),
])
def test_row_identity(N, K, gs, bits, dtype):
    """With mq.row_identity() a row has the bits of its own one-row call in every call of up
    to 32, kept sums or not; outside it the calls are as before."""
    g = _gen(1)
    banks = [bank(g, N, K, gs, bits, dtype)[0] for _ in range(2)]
    x = torch.randn((32, K), generator=g, device="cuda").to(dtype)
    kw = dict(group_size=gs, bits=bits)
    before = {M: mq.quantized_glu(x[:M], *banks, **kw) for M in (1, 24)}
    with mq.row_identity():
        one = torch.cat([mq.quantized_glu(x[m:m + 1], *banks, **kw) for m in range(32)])
        for M in (2, 3, 8, 15, 16, 17, 24, 31, 32):
            assert torch.equal(mq.quantized_glu(x[:M], *banks, **kw), one[:M])
        leaf = x[:20].clone().requires_grad_()
        assert torch.equal(mq.quantized_glu(leaf, *banks, **kw).detach(), one[:20])
    assert mq.set_row_identity(False) is False
    for M, h in before.items():
        assert torch.equal(mq.quantized_glu(x[:M], *banks, **kw), h)
    assert torch.equal(before[24], mq.quantized_glu(x[:24], *banks, **kw))


def test_row_identity_of_an_mlp():
    """Decode and verify of a whole MLP."""
    g = _gen(2)

    def layer(n, k):
        w = (torch.randn((n, k), generator=g, device="cuda") * k ** -0.5).to(BF)
        return QuantizedLinear.from_linear(w)
    mlp = QuantizedMLP(layer(4352, 1280), layer(4352, 1280), layer(1280, 4352))
    x = torch.randn((32, 1280), generator=g, device="cuda").to(BF)
    with mq.row_identity():
        one = torch.cat([mlp(x[m:m + 1]) for m in range(32)])
        for M in (2, 8, 16, 20, 32):
            assert torch.equal(mlp(x[:M]), one[:M])


def _layers(seed, **kw):
    g = _gen(seed)
    return [QuantizedLinear.from_linear((torch.randn((n, k), generator=g, device="cuda") * 0.05).to(BF),
                                        **kw) for n, k in ((192, 128), (192, 128), (128, 192))]


def _stepwise(mlp, x):
    gv, uv = mlp.gate_proj(x), mlp.up_proj(x)
    return mlp.down_proj((torch.nn.functional.silu(gv.float()) * uv.float()).to(gv.dtype))


class Adapted(torch.nn.Module):
    """A frozen layer and a low-rank adapter."""

    def __init__(self, base, rank=4):
        super().__init__()
        g = _gen(7)
        self.base = base
        self.a = torch.nn.Parameter(torch.randn((rank, base.input_dims), generator=g, device="cuda")
                                    .to(BF) * 0.1)
        self.b = torch.nn.Parameter(torch.randn((base.output_dims, rank), generator=g, device="cuda")
                                    .to(BF) * 0.1)

    def forward(self, x):
        return self.base(x) + x @ self.a.T @ self.b.T


class Doubled(QuantizedLinear):
    def forward(self, x):
        return 2 * super().forward(x)


class DoubledProduct(QuantizedLinear):
    def quantized_forward(self, x):
        return 2 * super().quantized_forward(x)


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("kind", ["adapter", "subclass", "product", "instance", "pre_hook", "hook",
                                  "global_hook", "routed"])
def test_mlp_calls_layers_that_are_not_plain(kind, which):
    """Gate or up wrapped, subclassed, hooked or routed: the MLP's result is of its call."""
    layers = _layers(3)
    x = torch.randn((40, 128), generator=_gen(4), device="cuda").to(BF)
    plain = QuantizedMLP(*layers)(x)
    layer, calls, handle = layers[which], [], None
    if kind == "adapter":
        layers[which] = Adapted(layer)
    elif kind in ("subclass", "product"):
        layer.__class__ = Doubled if kind == "subclass" else DoubledProduct
    elif kind == "instance":
        layer.forward = lambda v: 2 * QuantizedLinear.forward(layer, v)
    elif kind == "pre_hook":
        layer.register_forward_pre_hook(lambda m, a: (2 * a[0],))
    elif kind == "hook":
        layer.register_forward_hook(lambda m, a, y: 2 * y)
    elif kind == "global_hook":
        handle = torch.nn.modules.module.register_module_forward_hook(
            lambda m, a, y: 2 * y if m is layer else None)
    elif kind == "routed":
        mq.dispatch.enable(layer)
        seen = mq.dispatch.quantized_matmul
        mq.dispatch.quantized_matmul = lambda *a, **k: calls.append(1) or seen(*a, **k)
    try:
        mlp = QuantizedMLP(*layers)
        y = mlp(x)
        assert torch.equal(y, _stepwise(mlp, x))
        if kind == "routed":
            assert calls
        else:
            assert not torch.allclose(y.float(), plain.float(), rtol=0.05)
        if kind == "adapter":
            y.float().sum().backward()
            assert mlp.get_submodule(("gate_proj", "up_proj")[which]).b.grad.any()
    finally:
        if handle is not None:
            handle.remove()
        if kind == "routed":
            mq.dispatch.quantized_matmul = seen
    if kind in ("instance", "routed"):
        layer.__dict__.pop("forward", None)
        mq.dispatch.disable(layer)
        assert torch.equal(mlp(x), plain)


def test_mlp_under_the_class_patch():
    mlp = QuantizedMLP(*_layers(5))
    x = torch.randn((3, 128), generator=_gen(6), device="cuda").to(BF)
    plain = mlp(x)
    mq.dispatch.enable_class()
    try:
        assert torch.equal(mlp(x), _stepwise(mlp, x))
    finally:
        mq.dispatch.disable_class()
    assert torch.equal(mlp(x), plain)
