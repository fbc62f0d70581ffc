"""Forward-mode tangents through the products and the gated block."""

import pytest
import torch
from torch.autograd import forward_ad

import mlxturbo_amd as mq
from glu_helpers import activation, bank, check, matmul_ref
from mlxturbo_amd.nn import QQLinear, QuantizedLinear

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _pair(g, lead, K, dtype):
    return [torch.randn((*lead, K), generator=g, device="cuda").to(dtype) for _ in range(2)]


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("lead,bits,dtype", [((1,), 4, BF), ((2, 20), 8, HF), ((0,), 4, BF)])
def test_matmul(lead, bits, dtype, grad):
    g = _gen(1)
    b, w = bank(g, 72, 128, 64, bits, dtype)
    x, t = _pair(g, lead, 128, dtype)
    layer = QuantizedLinear(*b, bits=bits)
    want = layer(x)
    for f in (layer, lambda v: mq.quantized_matmul(v, *b, bits=bits)):
        with forward_ad.dual_level():
            y, ty = forward_ad.unpack_dual(f(forward_ad.make_dual(x.clone().requires_grad_(grad), t)))
            assert torch.equal(y, want) and y.requires_grad == grad
            assert torch.equal(ty, layer(t))
            # what has no tangent takes none
            assert forward_ad.unpack_dual(f(x)).tangent is None


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("M,dtype", [(1, BF), (9, HF), (40, BF)])
def test_glu(M, dtype, act, grad):
    g = _gen(2)
    (gate, wg), (up, wu) = (bank(g, 72, 128, 64, 4, dtype) for _ in range(2))
    x, t = _pair(g, (M,), 128, dtype)
    want = mq.quantized_glu(x, gate, up, act)
    with forward_ad.dual_level():
        h, th = forward_ad.unpack_dual(
            mq.quantized_glu(forward_ad.make_dual(x.clone().requires_grad_(grad), t), gate, up, act))
    assert torch.equal(h, want)
    gv, uv = x.double() @ wg.T, x.double() @ wu.T
    a, da = activation(gv, act)
    (tg, eg), (tu, eu) = (matmul_ref(t, w, dtype) for w in (wg, wu))
    # the tangents' products in their type; the float steps and the sums' error 2^-12 together
    off = da.abs() * uv.abs() * eg + a.abs() * eu
    off += 2.0 ** -12 * ((da.abs() + 0.1) * (uv.abs() + 0.1) * tg.abs() + (a.abs() + 0.1) * tu.abs())
    tan = da * tg * uv + a * tu
    check(th, tan, off + torch.finfo(dtype).eps / 2 * (tan.abs() + off) + 1e-7)


def test_mxfp4():
    g = _gen(3)
    w = (torch.randn((64, 128), generator=g, device="cuda") * 0.1).to(BF)
    x, t = _pair(g, (6,), 128, BF)
    layer = QuantizedLinear.from_linear(w, mode="mxfp4")
    with forward_ad.dual_level():
        y, ty = forward_ad.unpack_dual(layer(forward_ad.make_dual(x, t)))
        assert torch.equal(y, layer(x)) and torch.equal(ty, layer(t))
        with pytest.raises(NotImplementedError, match="qqmm"):
            QQLinear.from_linear(w)(forward_ad.make_dual(x, t))
