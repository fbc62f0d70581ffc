"""sample where a row's tiles, masses and lists are not the usual ones: more than 512 tiles,
tiles of more than 64 granules, masses of less than 2^-44 of the largest, and lists that
overflow in batches, whose listing and picking are launches of their own."""

import pytest
import torch

import mlxturbo_amd as mq
from test_gpu_sample import _check

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


# (a tile is 64 granules of 16 bytes, or as many as make 1024 tiles of a row)
@pytest.mark.parametrize("kw", [dict(temperature=0.8), dict(top_k=40), dict(top_k=600),
                                dict(top_k=900, top_p=0.9), dict(top_p=0.95), dict(min_p=0.02),
                                dict(top_k=3000, temperature=1.2), dict(temperature=0.0)], ids=str)
@pytest.mark.parametrize("R,V,dtype", [
    (1, 131073, F32),       # 513 tiles, the first number past the shorter bound's
    (2, 248320, F32),       # 970
    (17, 140001, F32),      # 547, in four launches
    (1, 262144, BF),        # 512, the last of it; masses of 2^-44
    (2, 262145, BF),        # 513 or 512; masses of 2^-43
    (1, 600007, HF),        # 128 granules a tile
    (2, 1100000, F32),      # 512 granules a tile; masses of 2^-41
])
def test_many_tiles(R, V, dtype, kw):
    g = _gen(V)
    logits = (torch.randn((R, V), generator=g, device="cuda") * 2.2).to(dtype)
    logits[:, 11::V // 300] += 6
    _check(logits, torch.rand(R, generator=g, device="cuda"), **kw)


@pytest.mark.parametrize("V,dtype", [(600007, BF), (1100003, F32)])
def test_many_tiles_at_odd_places(V, dtype):
    """A row that begins inside a granule, -inf in whole tiles, and one word alone."""
    g = _gen(1)
    logits = (torch.randn((3, V + 7), generator=g, device="cuda") * 2).to(dtype)[:, 3:V + 3]
    logits[1, V // 5:V // 2] = -float("inf")
    logits[2] = -float("inf")
    logits[2, V - 1] = -3
    u = torch.rand(3, generator=g, device="cuda")
    for kw in (dict(), dict(top_k=50), dict(top_p=0.9)):
        tok, lp = _check(logits, u, **kw)
        assert tok[2] == V - 1 and lp[2] == 0


def test_min_p_outside_its_range():
    """In a tensor: below 0 all, above 1 and NaN the first word alone, whatever else is set."""
    g = _gen(3)
    logits = (torch.randn((4, 5003), generator=g, device="cuda") * 2).to(BF)
    u = torch.full((4,), 0.97, device="cuda")
    m = torch.tensor([-0.5, 1.5, float("nan"), 0.0], device="cuda")
    for kw in (dict(), dict(top_k=50), dict(top_p=0.9)):
        tok, lp = mq.sample(logits, u, min_p=m, **kw)
        want, wlp = mq.sample(logits, u, **kw)
        top = logits.float().argmax(-1)
        assert tok.tolist() == [want[0], top[1], top[2], want[3]]
        assert lp[0] == wlp[0] and lp[1] == 0 and lp[2] == 0 and lp[3] == wlp[3]


OVERFLOWS = [
    dict(top_k=3), dict(top_k=60), dict(top_k=500), dict(top_k=11000), dict(top_k=33333),
    dict(top_p=0.31), dict(top_p=0.9137), dict(top_p=0.99999),
    dict(top_k=500, top_p=0.7713), dict(top_k=21000, top_p=0.6137), dict(top_k=60, top_p=0.5137),
    dict(top_p=0.9137, min_p=0.2), dict(top_k=21000, min_p=0.9), dict(top_k=700, temperature=0.5),
]


@pytest.mark.parametrize("kw", OVERFLOWS, ids=str)
@pytest.mark.parametrize("R,V,dtype", [(64, 40000, BF), (520, 5003, HF), (3, 20011, F32)])
def test_lists_that_overflow(R, V, dtype, kw):
    """Thousands of equal words at the cut: by radix over the row, from the bound of k, the
    bins of k and the bin of p.  Many rows list and pick in two launches (640 workgroups, and
    rows past the 256 of one sequence), few in one."""
    g = _gen(V)
    logits = torch.randint(0, 4, (R, V), generator=g, device="cuda").to(dtype)
    logits[R // 3] = 1.5
    logits[R // 2, :V // 2] = -float("inf")
    _check(logits, torch.rand(R, generator=g, device="cuda"), skip=0, **kw)


def test_overflow_beside_ordinary_rows():
    """Rows whose lists overflow do not change the others' results."""
    g = _gen(2)
    logits = (torch.randn((64, 40000), generator=g, device="cuda") * 2).to(BF)
    u = torch.rand(64, generator=g, device="cuda")
    for kw in (dict(top_k=50), dict(top_p=0.9), dict(top_k=2000, top_p=0.9)):
        want = mq.sample(logits, u, **kw)
        flat = logits.clone()
        flat[::5] = 0.25
        got = mq.sample(flat, u, **kw)
        rest = torch.arange(64, device="cuda") % 5 != 0
        assert all(torch.equal(a[rest], b[rest]) for a, b in zip(got, want))
        _check(flat, u, skip=0, **kw)
