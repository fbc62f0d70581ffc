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
