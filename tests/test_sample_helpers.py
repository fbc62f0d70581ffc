"""The sampling oracle on cases whose answers are known, and the refusals of sample and
of the gated block (CPU)."""

import numpy as np
import pytest
import torch

import mlxturbo_amd as mq
from mlxturbo_amd import _lib
from sample_helpers import INF, sample_row

FAKE = 256  # aligned, never dereferenced: validation fails before any HIP call


@pytest.fixture(scope="module")
def lib():
    import os
    if not os.path.exists(_lib.LIB_PATH):
        from mlxturbo_amd import build
        build.build()
    return _lib.lib()


def test_oracle_known_rows():
    l = np.log([0.1, 0.4, 0.2, 0.3])
    assert [sample_row(l, u)[0] for u in (0, 0.09, 0.11, 0.49, 0.51, 0.69, 0.71, 0.99)] == \
        [0, 0, 1, 1, 2, 2, 3, 3]
    assert sample_row(l, 0.99, temperature=0)[:2] == (1, 0.0)
    # k = 2: words 1 and 3; 4/7 of the mass is word 1's
    assert [sample_row(l, u, top_k=2)[0] for u in (0.57, 0.58)] == [1, 3]
    assert sample_row(l, 0.6, top_k=2)[1] == pytest.approx(np.log(3 / 7))
    # p: the words before which the mass is below it, in order 1, 3, 2, 0
    assert [sample_row(l, 0.999, top_p=p)[0] for p in (0.39, 0.41, 0.71, 0.91)] == [1, 3, 3, 3]
    assert [sample_row(l, 0.0, top_p=p)[0] for p in (0.39, 0.41, 0.71, 0.91)] == [1, 1, 1, 0]
    assert [sample_row(l, 0.0, min_p=p)[0] for p in (0.2, 0.3, 0.6)] == [0, 1, 1]
    # ties go to the lowest index
    assert [sample_row([1, 1, 1, 1], u, top_k=2)[0] for u in (0.4, 0.6)] == [0, 1]
    assert sample_row([-INF, float("nan")], 0.5) == (-1, -INF, INF)


def test_sample_runs_on_the_gpu_only():
    with pytest.raises(ValueError, match="GPU only"):
        mq.sample(torch.zeros(2, 8), torch.zeros(2))
    with pytest.raises(ValueError, match="GPU only"):
        mq.quantized_glu(torch.zeros(1, 64, dtype=torch.bfloat16),
                         *[(torch.zeros(8, 8, dtype=torch.int32), torch.zeros(8, 1), torch.zeros(8, 1))] * 2)


def test_activation_and_format_refusals():
    with pytest.raises(ValueError, match="activation"):
        mq.quantized_glu(torch.zeros(1), (), (), "relu")
    with pytest.raises(ValueError, match="mxfp4"):
        mq.quantized_glu(torch.zeros(1), (), (), mode="mxfp4", bits=8)
    with pytest.raises(ValueError, match="w, scales, biases"):
        mq.quantized_glu(torch.zeros(1), (1, 2), (1, 2, 3))


def _sample(lib, **kw):
    a = dict(logits=FAKE, stride=100, R=2, V=100, dtype=0, u=FAKE, tokens=FAKE, logprobs=FAKE,
             ws=FAKE, bytes=1 << 30)
    a.update(kw)
    return lib.mq_sample(a["logits"], a["stride"], a["R"], a["V"], a["dtype"], a["u"], None, 1.0,
                         None, 0, None, 1.0, None, 0.0, a["tokens"], a["logprobs"], a["ws"],
                         a["bytes"], None)


@pytest.mark.parametrize("kw,code,needle", [
    (dict(logits=None), -1, "non-null"),
    (dict(u=None), -1, "non-null"),
    (dict(tokens=None), -1, "non-null"),
    (dict(logprobs=None), -1, "non-null"),
    (dict(dtype=5), -1, "dtype"),
    (dict(R=-1), -1, "rows"),
    (dict(V=0), -1, "vocabulary"),
    (dict(stride=-100), -1, "row_stride"),
    (dict(V=(1 << 30) + 1), -2, "2^30"),
    (dict(logits=FAKE + 1), -1, "aligned"),
    (dict(logits=FAKE + 2, dtype=2), -1, "aligned"),
    (dict(ws=None), -1, "workspace"),
    (dict(ws=FAKE + 8), -1, "workspace"),
    (dict(bytes=100), -1, "workspace"),
])
def test_sample_argument_validation(lib, kw, code, needle):
    assert _sample(lib, **kw) == code
    assert needle in lib.mq_last_error().decode()


def test_sample_no_rows(lib):
    assert _sample(lib, R=0) == 0
    assert lib.mq_sample_workspace_size(0, 100) == 0
    # rows of a sequence share their workspace
    assert lib.mq_sample_workspace_size(256, 5000) == lib.mq_sample_workspace_size(9999, 5000) > 0


def _glu(lib, name="mq_quantized_glu", **kw):
    a = dict(x=FAKE, w=FAKE, s=FAKE, b=FAKE, w2=FAKE, s2=FAKE, b2=FAKE, out=FAKE, g=None, u=None,
             M=4, N=100, K=256, gs=64, bits=4, dtype=0, act=0, ws=None, bytes=0)
    a.update(kw)
    banks = [a[k] for k in ("w", "s", "b", "w2", "s2", "b2")]
    tail = [a[k] for k in ("M", "N", "K", "gs", "bits", "dtype", "act", "ws", "bytes")] + [None]
    if name == "mq_quantized_glu":
        return lib.mq_quantized_glu(a["x"], *banks, a["out"], a["g"], a["u"], *tail)
    return lib.mq_quantized_glu_grad(a["x"], a["g"], a["u"], *banks, a["out"], *tail)


COMMON = [
    (dict(x=None), -1, "non-null"),
    (dict(out=None), -1, "non-null"),
    (dict(w2=None), -1, "non-null"),
    (dict(b=None), -1, "biases"),
    (dict(b2=None), -1, "biases"),
    (dict(gs=48), -1, "group_size"),
    (dict(bits=6), -2, "no matmul kernel"),
    (dict(K=100), -1, "multiple"),
    (dict(dtype=2), -2, "float32"),
    (dict(act=2), -1, "activation"),
    (dict(x=FAKE + 2), -1, "aligned"),
    (dict(w2=FAKE + 4), -1, "aligned"),
    (dict(ws=FAKE + 8, bytes=1 << 20), -1, "aligned"),
    (dict(M=-1), -1, "M=-1"),
    (dict(N=1 << 31), -1, "N="),
    (dict(K=1 << 28), -1, "K="),
]


@pytest.mark.parametrize("kw,code,needle", COMMON + [(dict(g=FAKE), -1, "together")])
def test_glu_argument_validation(lib, kw, code, needle):
    assert _glu(lib, **kw) == code
    assert needle in lib.mq_last_error().decode()


@pytest.mark.parametrize("kw,code,needle", COMMON + [
    (dict(g=None), -1, "gate_sums"),
    (dict(), -1, "workspace"),
    (dict(N=0), -2, "no columns"),
    (dict(N=1 << 30, K=128), -2, "31-bit"),
    (dict(N=1 << 22, K=64), -2, "31-bit"),
])
def test_glu_grad_argument_validation(lib, kw, code, needle):
    assert _glu(lib, "mq_quantized_glu_grad", **{"g": FAKE, "u": FAKE, **kw}) == code
    assert needle in lib.mq_last_error().decode()


def _matmul_grad(lib, d=FAKE, w=FAKE, N=128, K=256, bits=4):
    return lib.mq_quantized_matmul_grad(d, w, FAKE, FAKE, FAKE, 4, N, K, 64, bits, 0, None, 0, None)


@pytest.mark.parametrize("kw,code,needle", [
    (dict(d=None), -1, "non-null"), (dict(w=None), -1, "non-null"),
    (dict(bits=3), -2, "no matmul kernel"), (dict(N=0), -2, "no columns"),
    (dict(d=FAKE + 2), -1, "aligned"), (dict(N=1 << 26), -2, "31-bit"),
    (dict(N=100), -1, "workspace"),
])
def test_matmul_grad_argument_validation(lib, kw, code, needle):
    assert _matmul_grad(lib, **kw) == code
    assert needle in lib.mq_last_error().decode()


def test_grad_workspace_sizes(lib):
    # rows padded to whole steps of 64 columns; the block's two halves
    assert lib.mq_quantized_matmul_grad_workspace_size(4, 100, 256, 64, 4) >= 4 * 128 * 2
    assert lib.mq_quantized_glu_grad_workspace_size(4, 100, 256, 64, 4) >= 4 * 256 * 2
    assert lib.mq_quantized_glu_workspace_size(16, 17408, 5120, 64, 4) == 0
