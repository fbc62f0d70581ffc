"""sample against the definition (sample_helpers.py): every path, at the masks,
ties, settings and strides where it can go wrong.

Tokens are equal where u's place and the cuts are further than 2^-30 of the kept mass
from a word's end (the kernel's masses are rounded to 2^-44 of the largest, 2^-45
each, so sums over 2^18 words are off by 2^-27 at most and by about 2^-37 as they
round; a test whose margin is smaller says nothing and is left out, which the tests bound).
Log probabilities: the float rounding, and the masses' error over a kept mass of at
least one."""

import math

import numpy as np
import pytest
import torch

import mlxturbo_amd as mq
from sample_helpers import INF, sample_row

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rows(v, n):
    return v.tolist() if isinstance(v, torch.Tensor) else [v] * n


def _check(logits, u, skip=0.02, **kw):
    before = mq.launch_count()
    tok, lp = mq.sample(logits, u, **kw)
    assert mq.launch_count() > before
    assert tok.dtype == torch.int32 and lp.dtype == torch.float32
    assert tok.shape == lp.shape == logits.shape[:-1]
    V = logits.shape[-1]
    l = logits.reshape(-1, V).float().cpu().numpy()
    n = l.shape[0]
    keys = ("temperature", "top_k", "top_p", "min_p")
    base = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0}
    sets = [_rows({**base, **kw}[k], n) for k in keys]
    got, glp, us = tok.reshape(-1).tolist(), lp.reshape(-1).tolist(), u.reshape(-1).tolist()
    out = 0
    for r in range(n):
        want, wlp, margin = sample_row(l[r], us[r], *[s[r] for s in sets])
        if margin < 2.0 ** -30:
            out += 1
            continue
        where = f"row {r}, {dict(zip(keys, [s[r] for s in sets]))}, u {us[r]}"
        assert got[r] == want, where
        if math.isinf(wlp):
            assert glp[r] == wlp, where
        else:
            assert abs(glp[r] - wlp) <= 2.0 ** -24 * abs(wlp) + 2.0 ** -27, where
    assert out <= max(1, skip * n), f"{out} of {n} rows at a border"
    return tok, lp


SETTINGS = [
    dict(),
    dict(temperature=0.0),
    dict(temperature=0.7),
    dict(top_k=1),
    dict(top_k=40, temperature=1.3),
    dict(top_p=0.9),
    dict(top_p=0.95, temperature=0.6),
    dict(min_p=0.05),
    dict(top_k=50, top_p=0.9, min_p=0.02, temperature=0.8),
    dict(top_p=0.5, min_p=0.2),
    dict(top_k=10 ** 6, top_p=0.99),
    dict(top_p=0.0),
]


@pytest.mark.parametrize("kw", SETTINGS, ids=str)
@pytest.mark.parametrize("R,V,dtype", [(1, 1, F32), (2, 7, BF), (3, 63, HF), (5, 1000, F32),
                                       (4, 2049, BF), (3, 32000, HF), (2, 151937, BF)])
def test_settings(R, V, dtype, kw):
    g = _gen(V)
    logits = (torch.randn((R, V), generator=g, device="cuda") * 3).to(dtype)
    _check(logits, torch.rand(R, generator=g, device="cuda"), **kw)


@pytest.mark.parametrize("R,V", [(300, 5003), (64, 40000), (17, 248320)])
def test_rows_of_their_own(R, V):
    g = _gen(R)
    cu = "cuda"
    logits = (torch.randn((R, V), generator=g, device=cu) * 2.5).to(BF)
    logits[:, ::97] += 4
    logits[R // 2, V // 3:] = -INF
    kw = dict(temperature=torch.rand(R, generator=g, device=cu) * 1.5,
              top_k=torch.randint(-1, 300, (R,), generator=g, device=cu),
              top_p=torch.rand(R, generator=g, device=cu) * 1.2,
              min_p=torch.rand(R, generator=g, device=cu) * 0.1)
    kw["temperature"][::7] = 0
    kw["top_p"] = kw["top_p"].clamp(max=1)
    _check(logits, torch.rand(R, generator=g, device=cu), **kw)


@pytest.mark.parametrize("kw", SETTINGS, ids=str)
def test_ties(kw):
    """Few distinct values: cuts fall among equal logits, the lower index first; and lists
    of more than 4096 equal words."""
    g = _gen(3)
    logits = torch.randint(0, 4, (6, 20011), generator=g, device="cuda").to(BF)
    logits[3] = 1.5                                   # all equal
    logits[4, :-5] = -INF
    _check(logits, torch.rand(6, generator=g, device="cuda"), **kw)


@pytest.mark.parametrize("k", [1, 4095, 4096, 4097, 20000, 30000])
@pytest.mark.parametrize("top_p", [1.0, 0.8])
def test_long_lists(k, top_p):
    g = _gen(4)
    logits = (torch.randn((2, 30000), generator=g, device="cuda") * 1.5).to(HF)
    _check(logits, torch.rand(2, generator=g, device="cuda"), top_k=k, top_p=top_p)


@pytest.mark.parametrize("kw", SETTINGS, ids=str)
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_masked_and_special(dtype, kw):
    V = 3001
    g = _gen(5)
    big = torch.finfo(dtype)
    l = (torch.randn((9, V), generator=g, device="cuda") * 2).to(dtype)
    l[0] = -INF                                       # nothing
    l[1] = float("nan")
    l[2] = -INF
    l[2, 1234] = -5                                   # one word
    l[3, ::2] = float("nan")
    l[4, 5] = INF                                     # all the mass
    l[5, [7, 9]] = INF                                # shared
    l[6] = big.min                                    # the type's lowest value as a mask
    l[6, 100:110] = 1
    l[7] = big.min                                    # nothing but that
    l[8, 17] = big.max
    u = torch.rand(9, generator=g, device="cuda")
    # (rows 5 and 6, of two and of ten equal words, have top_p = 0.5 at a word's end)
    tok, lp = _check(l, u, skip=2 / 9, **kw)
    assert tok[0] == -1 and tok[1] == -1 and lp[0] == -INF and tok[2] == 1234


def test_ends_of_u():
    """0 takes the first word of mass, the largest float below 1 and what lies outside
    [0, 1) a word inside the row."""
    l = torch.tensor([-INF, 1.0, 2.0, -200.0, 0.5, -INF], device="cuda").repeat(6, 1)
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, 7.0, -3.0, float("nan")], device="cuda")
    for kw in (dict(), dict(top_k=4), dict(top_p=0.999)):
        tok, _ = mq.sample(l, u, **kw)
        assert tok.tolist() == [1, 4, 4, 4, 1, 1]


@pytest.mark.parametrize("kw", [dict(temperature=0.7), dict(top_k=30), dict(top_p=0.9)], ids=str)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_strides(dtype, kw):
    """Rows inside a longer buffer, at odd places, three dimensions, a transposed one."""
    g = _gen(6)
    big = (torch.randn((4, 3, 5003), generator=g, device="cuda") * 2).to(dtype)
    u = torch.rand(4, generator=g, device="cuda")
    u3 = torch.rand((4, 3), generator=g, device="cuda")
    for l, v in ((big[:, -1], u), (big[:, 1, 3:4098], u), (big, u3), (big[:, :, 1:-1], u3),
                 (big.transpose(0, 1), u3.t()), (big[0].t().contiguous().t(), u3[0]),
                 (big[:1, 0].expand(4, 5003), u), (big[0, 0], u[0])):
        want = mq.sample(l.contiguous(), v.contiguous(), **kw)
        got = mq.sample(l, v, **kw)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    _check(big[:, 1, 3:4098], u, **kw)


def test_rows_do_not_depend_on_the_batch():
    g = _gen(7)
    l = (torch.randn((40, 50257), generator=g, device="cuda") * 2).to(BF)
    u = torch.rand(40, generator=g, device="cuda")
    for kw in (dict(), dict(top_k=100), dict(top_p=0.9)):
        tok, lp = mq.sample(l, u, **kw)
        for r in (0, 17, 39):
            t1, p1 = mq.sample(l[r:r + 1], u[r:r + 1], **kw)
            assert torch.equal(t1, tok[r:r + 1]) and torch.equal(p1, lp[r:r + 1])


def test_graph_and_streams():
    """A captured call, replayed between eager ones on another stream."""
    g = _gen(8)
    l = (torch.randn((8, 32000), generator=g, device="cuda") * 2).to(BF)
    u = torch.rand(8, generator=g, device="cuda")
    kw = dict(temperature=0.8, top_k=torch.tensor([0, 5, 0, 40, 0, 7, 0, 1], device="cuda"),
              top_p=torch.tensor([1, 1, 0.9, 0.5, 1, 1, 0.3, 1.0], device="cuda"))
    mq.sample(l, u, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tok, lp = mq.sample(l, u, **kw)
    side = torch.cuda.Stream()
    for i in range(4):
        l.copy_((torch.randn(l.shape, generator=g, device="cuda") * 2).to(BF))
        u.copy_(torch.rand(8, generator=g, device="cuda"))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            other = mq.sample(l.flip(0), u, **kw)
        graph.replay()
        torch.cuda.synchronize()
        want = mq.sample(l, u, **kw)
        assert torch.equal(tok, want[0]) and torch.equal(lp, want[1])
        assert torch.equal(other[0], mq.sample(l.flip(0), u, **kw)[0])


def test_head_then_sample():
    """A quantized head's logits of drafted positions, as they are used."""
    from mlxturbo_amd.nn import QuantizedLinear
    g = _gen(9)
    w = (torch.randn((50257, 512), generator=g, device="cuda") * 0.05).to(BF)
    head = QuantizedLinear.from_linear(w, bits=8)
    x = torch.randn((2, 5, 512), generator=g, device="cuda").to(BF)
    logits = head(x)
    _check(logits, torch.rand((2, 5), generator=g, device="cuda"), top_k=64, top_p=0.95)
    tok, _ = mq.sample(logits, torch.zeros((2, 5), device="cuda"), temperature=0)
    assert torch.equal(tok.long(), logits.float().argmax(-1))


@pytest.mark.parametrize("dtype,spread", [(F32, 0.012), (F32, 1e-5), (F32, 0.0), (BF, 0.012),
                                          (HF, 0.3), (HF, 0.012)])
@pytest.mark.parametrize("V", [2, 600, 3001, 4096, 4099])
@pytest.mark.parametrize("kw", [dict(top_p=p, min_p=m) for p in (1e-6, 0.0377, 0.5137, 0.999)
                                for m in (0.0, 0.993)], ids=str)
def test_cut_of_p_inside_one_bin(V, dtype, spread, kw):
    """The cut of p among thousands of words of nearly, or just, the same logit, some with
    masked words and larger ones between them."""
    g = _gen(V)
    logits = 1 + torch.rand((3, V), generator=g, device="cuda") * spread
    logits[1, ::3] = -INF
    if V > 10:
        logits[2, 5::7] += 2
    # (these p times counts of equal words are no whole numbers; a row in three may lie at a
    # border by u)
    _check(logits.to(dtype), torch.rand(3, generator=g, device="cuda"), skip=1 / 3, **kw)
