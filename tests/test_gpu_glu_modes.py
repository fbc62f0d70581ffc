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
