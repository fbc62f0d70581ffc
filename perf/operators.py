"""Performance cases of the MXFP4 operators: quantization, and products with MXFP4 weights.

MXFP4 (OCP Microscaling formats v1.0): groups of 32 values along the last axis
share one power of two, 2^(e - 127) with e a byte (255: NaN); a value is a 4-bit
E2M1 code (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign) times it.  Codes are packed
eight to a uint32 word, low bits first.  A case is one call of

* ``roundtrip``: ``mq.quantize`` then ``mq.dequantize`` of a weight matrix, what
  a layer's weights become when it is moved to the format;
* ``qmm``: ``mq.quantized_matmul``, a layer over MXFP4 weights;
* ``gather``: ``mq.gather_qmm``, one projection of a mixture of experts: every
  token through its top-k experts' matrices;
* ``qqmm``: ``mq.qqmm``, a layer that brings its activations into MXFP4 as well
  and multiplies in 4 bits.

The plain forms dequantize to float32 and multiply there.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_MODE = "mxfp4"


def listed():
    return [
        # One expert's matrix brought into the format, from a float32 master.
        {"name": "roundtrip_512x2048_fp32", "kind": "roundtrip", "N": 512, "K": 2048,
         "dtype": "fp32"},
        # Loading: the MLP matrix of a 27B-class model.
        {"name": "roundtrip_17408x5120", "kind": "roundtrip", "N": 17408, "K": 5120,
         "dtype": "bf16"},
        # The smallest product: one attention projection for one decoded token.
        {"name": "qmm_m1_4096x4096", "kind": "qmm", "M": 1, "N": 4096, "K": 4096, "dtype": "bf16"},
        # A speculative-verify step of 8 drafted tokens through an MLP matrix.
        {"name": "qmm_m8_17408x5120", "kind": "qmm", "M": 8, "N": 17408, "K": 5120,
         "dtype": "bf16"},
        # A decode batch of 45 sequences, the down projection, in fp16.
        {"name": "qmm_m45_5120x17408_fp16", "kind": "qmm", "M": 45, "N": 5120, "K": 17408,
         "dtype": "fp16"},
        # A prefill chunk of 2048 tokens.
        {"name": "qmm_m2048_17408x5120", "kind": "qmm", "M": 2048, "N": 17408, "K": 5120,
         "dtype": "bf16"},
        # One decoded token through its 8 of 512 experts.
        {"name": "gather_t1_e512", "kind": "gather", "T": 1, "k": 8, "E": 512, "N": 512, "K": 2048,
         "dtype": "bf16", "zipf": True},
        # A ragged prompt over 128 experts, evenly spread, fp16.
        {"name": "gather_t301_e128_fp16", "kind": "gather", "T": 301, "k": 8, "E": 128, "N": 768,
         "K": 2048, "dtype": "fp16", "zipf": False},
        # A prefill chunk over 512 experts, skewed: most see a few rows, some thousands.
        {"name": "gather_t2048_e512", "kind": "gather", "T": 2048, "k": 8, "E": 512, "N": 512,
         "K": 2048, "dtype": "bf16", "zipf": True},
        # Four verified tokens through a layer with 4-bit activations.
        {"name": "qqmm_m4_17408x5120", "kind": "qqmm", "M": 4, "N": 17408, "K": 5120,
         "dtype": "bf16"},
        # An odd prompt through the down projection.
        {"name": "qqmm_m509_5120x17408", "kind": "qqmm", "M": 509, "N": 5120, "K": 17408,
         "dtype": "fp16"},
        # The largest: a prefill chunk of 4096 tokens.
        {"name": "qqmm_m4096_17408x5120", "kind": "qqmm", "M": 4096, "N": 17408, "K": 5120,
         "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: every size log-uniform, inner dimensions in whole groups
    of 32, row counts any."""
    c = {"kind": rng.choice(["roundtrip", "qmm", "qmm", "qmm", "gather", "gather", "qqmm",
                             "qqmm"]),
         "dtype": rng.choice(["bf16", "bf16", "fp16"])}
    if c["kind"] == "gather":
        c["E"] = _log(rng, 8, 512)
        c["k"] = rng.randint(1, 8)
        c["N"] = _log(rng, 200, 1500)
        c["K"] = 32 * _log(rng, 512 / 32, 2560 / 32)
        c["T"] = _log(rng, 1, 2048)
        c["zipf"] = rng.random() < 0.5
        return c
    c["K"] = 32 * _log(rng, 1024 / 32, 17408 / 32)
    c["N"] = _log(rng, 512, 17408)
    if c["kind"] == "roundtrip":
        c["N"] = min(c["N"], 5120 * 17408 // c["K"])
        c["dtype"] = rng.choice(["bf16", "fp16", "fp32"])
    else:
        most = 2048 if c["kind"] == "qmm" else 4096
        c["M"] = _log(rng, 1, most * min(1.0, 5120 * 17408 / (c["K"] * c["N"])))
    return c


# ---- inputs -----------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _pow2(p):
    """2^p in float32, p whole and in -127..127: from the bits, exactly."""
    return torch.where(p < -126, 2.0 ** -127, ((p + 127).clamp_min(1) << 23).view(torch.float32))


def _mx_codes(v):
    """float32 ``(..., K)`` -> (E2M1 codes int32 ``(..., K)``, scale bytes int32
    ``(..., K / 32)``): the scale is the largest magnitude's power of two over
    4 (E2M1's largest power), codes are rounded to nearest, ties to even, and
    saturate at 6.  A group that holds a NaN or an infinity is NaN: byte 255."""
    v = v.reshape(*v.shape[:-1], -1, 32)
    top = v.abs().amax(-1, keepdim=True)
    field = (top.view(torch.int32) >> 23) & 255       # floor(log2) + 127
    e = (field - 2).clamp_min(0)
    q = v * _pow2(127 - e)
    a = q.abs()
    code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int()
            + (a > 2.5).int() + (a >= 3.5).int() + (a > 5).int())
    code = code + 8 * torch.signbit(q).int()
    bad = field == 255
    code, e = torch.where(bad, 0, code), torch.where(bad, 255, e)
    return code.reshape(*code.shape[:-2], -1), e.squeeze(-1)


def _mx_values(code, e):
    """What codes and scale bytes stand for, in float32."""
    m = code & 7
    a = torch.where(m < 2, m * 0.5, (1 + 0.5 * (m & 1)) * _pow2((m >> 1) - 1))
    a = torch.where(code > 7, -a, a)
    s = torch.where(e == 255, math.nan, _pow2(e.clamp_max(254) - 127))
    return (a.reshape(*e.shape, 32) * s.unsqueeze(-1)).reshape(a.shape)


def _unpack(w):
    """uint32 words -> codes int32."""
    b = w.view(torch.uint8)
    return torch.stack([b & 15, b >> 4], dim=-1).reshape(*b.shape[:-1], -1).int()


def _weights(g, *shape):
    """N(0, 0.02) matrices as an MXFP4 checkpoint holds them: (uint32 words,
    uint8 scales)."""
    rows, K = math.prod(shape[:-1]), shape[-1]
    w = torch.empty((rows, K // 2), dtype=torch.uint8, device="cuda")
    s = torch.empty((rows, K // 32), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 27) // K)
    for r in range(0, rows, step):
        n = min(step, rows - r)
        code, e = _mx_codes(torch.randn((n, K), generator=g, device="cuda").mul_(0.02))
        w[r:r + n] = (code[:, 0::2] | (code[:, 1::2] << 4)).to(torch.uint8)
        s[r:r + n] = e.to(torch.uint8)
    return (w.view(torch.int32).view(torch.uint32).reshape(*shape[:-1], K // 8),
            s.reshape(*shape[:-1], K // 32))


def _routing(g, c):
    """Top-k experts of each token, Zipf-distributed over the experts or even
    (Gumbel perturbation: draws without replacement)."""
    E = c["E"]
    p = torch.zeros(E, device="cuda")
    if c["zipf"]:
        p = -1.1 * torch.arange(1, E + 1, device="cuda", dtype=torch.float32).log()
        p = p[torch.randperm(E, generator=g, device="cuda")]
    u = torch.rand((c["T"], E), generator=g, device="cuda").clamp_(1e-7, 1 - 1e-7)
    return (p - torch.log(-torch.log(u))).topk(c["k"], dim=-1).indices.int()


def prepare(case, seed):
    """What a program holds before the call: the layer's weights and the step's
    activations and routing."""
    c, g = case, _gen(seed)
    dt = _DTYPES[c["dtype"]]
    state = {"kind": c["kind"]}
    if c["kind"] == "roundtrip":
        state["w"] = torch.randn((c["N"], c["K"]), generator=g, device="cuda").mul_(0.02).to(dt)
        return state
    if c["kind"] == "gather":
        state["w"], state["s"] = _weights(g, c["E"], c["N"], c["K"])
        state["x"] = torch.randn((c["T"], 1, 1, c["K"]), generator=g, device="cuda").to(dt)
        state["idx"] = _routing(g, c)
        return state
    state["w"], state["s"] = _weights(g, c["N"], c["K"])
    state["x"] = torch.randn((c["M"], c["K"]), generator=g, device="cuda").to(dt)
    return state


# ---- one pass ---------------------------------------------------------------

def _plain_gather(x, w, s, idx):
    """x (T, 1, 1, K), idx (T, k) -> (T, k, 1, N), in float32."""
    (T, k), (E, N), K = idx.shape, w.shape[:2], x.shape[-1]
    flat, P = idx.reshape(-1).long(), idx.numel()
    rows = x.reshape(T, K).float().repeat_interleave(k, 0)
    if P <= 64:
        deq = _mx_values(_unpack(w.view(torch.int32)[flat]), s[flat].int())
        return torch.matmul(deq, rows.unsqueeze(-1)).reshape(T, k, 1, N)
    # each expert's rows side by side, padded to the largest count
    order = torch.argsort(flat, stable=True)
    count = torch.bincount(flat, minlength=E)
    most = int(count.max())
    e = flat[order]
    place = e * most + torch.arange(P, device=e.device) - (count.cumsum(0) - count)[e]
    padded = torch.zeros((E * most, K), device=x.device)
    padded[place] = rows[order]
    deq = _mx_values(_unpack(w.view(torch.int32)), s.int())
    y = torch.matmul(padded.reshape(E, most, K), deq.transpose(1, 2).contiguous())
    out = torch.empty((P, N), device=x.device)
    out[order] = y.reshape(E * most, N)[place]
    return out.reshape(T, k, 1, N)


def run(state):
    """One call, or its plain form."""
    kind, w = state["kind"], state["w"]
    if own:
        import mlxturbo_amd as mq
        if kind == "roundtrip":
            wq, s = mq.quantize(w, mode=_MODE)
            return mq.dequantize(wq, s, mode=_MODE, dtype=w.dtype)
        if kind == "qmm":
            return mq.quantized_matmul(state["x"], w, state["s"], mode=_MODE)
        if kind == "gather":
            return mq.gather_qmm(state["x"], w, state["s"], rhs_indices=state["idx"], mode=_MODE)
        return mq.qqmm(state["x"], w, state["s"], mode=_MODE)
    if kind == "roundtrip":
        return _mx_values(*_mx_codes(w.float())).to(w.dtype)
    x, s = state["x"], state["s"]
    if kind == "gather":
        return _plain_gather(x, w, s, state["idx"]).to(x.dtype)
    xf = x.float()
    if kind == "qqmm":
        xf = _mx_values(*_mx_codes(xf))
    deq = _mx_values(_unpack(w.view(torch.int32)), s.int())
    return torch.matmul(xf, deq.T).to(x.dtype)


# ---- what a pass needs ------------------------------------------------------

_BITS = {"bf16": 16, "fp16": 16, "fp32": 32}


def _bank(n):
    """Bytes of n values in the format."""
    return n / 2 + n / 32


def _experts(c):
    """Distinct experts that T tokens of k are expected to reach."""
    E, k, T = c["E"], min(c["k"], c["E"]), c["T"]
    p = [r ** -1.1 if c["zipf"] else 1.0 for r in range(1, E + 1)]
    t = sum(p)
    return max(k, sum(1 - (1 - min(1.0, k * v / t)) ** T for v in p))


def work(case):
    c, N, K = case, case["N"], case["K"]
    size = _BITS[c["dtype"]] // 8
    if c["kind"] == "roundtrip":
        # the codes are written and read again: two calls
        return {"bytes": 2 * N * K * size + 2 * _bank(N * K), "flops": 4 * N * K}
    if c["kind"] == "gather":
        T, k = c["T"], c["k"]
        return {"bytes": _experts(c) * _bank(N * K) + 2 * T * K + 4 * T * k + 2 * T * k * N,
                "flops": 2 * T * k * N * K}
    M = c["M"]
    return {"bytes": _bank(N * K) + 2 * M * (K + N), "flops": 2 * M * N * K}


# ---- the same in 64 bits ----------------------------------------------------

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _pow2_64(p):
    return ((p.long() + 1023) << 52).view(torch.float64)


def _deq64(w, s):
    """The values of packed codes, by table, in float64 (finite scales)."""
    b = w.view(torch.int32).view(torch.uint8).long()
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), dtype=torch.float64, device=b.device)
    v = torch.stack([table[b % 16], table[b // 16]], dim=-1).reshape(*s.shape, 32)
    return (v * _pow2_64(s.long() - 127).unsqueeze(-1)).reshape(*s.shape[:-1], -1)


def _round64(v):
    """Every value's nearest in its group's format, in float64."""
    q = v.double().reshape(*v.shape[:-1], -1, 32)
    top = q.abs().amax(-1, keepdim=True)
    # frexp: top = f 2^p with f in [1/2, 1), so floor(log2(top)) = p - 1
    p = _pow2_64(torch.where(top == 0, -126, (torch.frexp(top).exponent - 3).clamp_min(-127)))
    a = q.abs() / p
    grid = torch.tensor(_E2M1, dtype=torch.float64, device=q.device)
    mid = (grid[1:] + grid[:-1]) / 2
    i = torch.searchsorted(mid, a.contiguous())           # midpoints below a
    tie = (i < 7) & (a == mid[i.clamp_max(6)]) & (i % 2 == 1)
    i = i + tie
    return (torch.copysign(grid[i], q) * p).reshape(v.shape)


def exact(case, seed):
    """`run` on the same inputs in float64."""
    d = prepare(case, seed)
    if case["kind"] == "roundtrip":
        return _round64(d["w"])
    if case["kind"] != "gather":
        x = d["x"].double() if case["kind"] == "qmm" else _round64(d["x"])
        step = max(1, (1 << 26) // case["K"])
        return torch.cat([x @ _deq64(d["w"].view(torch.int32)[r:r + step], d["s"][r:r + step]).T
                          for r in range(0, case["N"], step)], dim=-1)
    T, k = d["idx"].shape
    x, idx = d["x"].reshape(T, -1).double(), d["idx"]
    out = torch.empty((T, k, case["N"]), dtype=torch.float64, device=x.device)
    for e in torch.unique(idx).tolist():
        t, j = (idx == e).nonzero(as_tuple=True)
        out[t, j] = x[t] @ _deq64(d["w"].view(torch.int32)[e], d["s"][e]).T
    return out.unsqueeze(-2)
