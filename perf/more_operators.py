"""Performance cases of the dense gated feed-forward block, of products trained through, and of sampling.

What a dense model needs around the products that it has: the first half of its
feed-forward block, gradients past its frozen weights, and a token from the
head's logits.  A case is one call, or one training step, of

* ``glu``: ``mq.quantized_glu``, ``act(x Wg^T) * (x Wu^T)`` over the block's gate
  and up matrices;
* ``glu_train``: the same with x's gradient from h's, as adapters below the
  block are trained;
* ``qmm_train``: ``mq.quantized_matmul`` with x's gradient, a down projection or
  a head in such a step;
* ``sample``: ``mq.sample``, a token for each row of logits from a given uniform
  number: temperature, the k largest, the most probable of mass p, and no less
  probable than min_p of the most probable.

Weights are affine codes of 4 or 8 bits, low bits first in uint32 words, with a
scale and a bias per group along K; a weight is ``T(scale * code + bias)`` in the
layer's type T.  The plain forms make the weights and multiply in float32; they
sample in float64, where probabilities meet a border.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # One decoded token through the MLP of a 27B-class model.
        {"name": "glu_m1_17408x5120", "kind": "glu", "M": 1, "N": 17408, "K": 5120, "gs": 64,
         "bits": 4, "act": "silu", "dtype": "bf16"},
        # A speculative-verify step of 8 drafted tokens.
        {"name": "glu_m8_17408x5120", "kind": "glu", "M": 8, "N": 17408, "K": 5120, "gs": 64,
         "bits": 4, "act": "silu", "dtype": "bf16"},
        # A decode batch of 45 sequences, 8-bit codes, odd width, fp16, the tanh GELU.
        {"name": "glu_m45_9001x2560_b8_fp16", "kind": "glu", "M": 45, "N": 9001, "K": 2560,
         "gs": 128, "bits": 8, "act": "gelu_tanh", "dtype": "fp16"},
        # A prefill chunk of 2048 tokens.
        {"name": "glu_m2048_17408x5120", "kind": "glu", "M": 2048, "N": 17408, "K": 5120,
         "gs": 64, "bits": 4, "act": "silu", "dtype": "bf16"},
        # A training step of one short, ragged sequence, small groups.
        {"name": "glu_train_m301_8192x2048", "kind": "glu_train", "M": 301, "N": 8192, "K": 2048,
         "gs": 32, "bits": 4, "act": "gelu_tanh", "dtype": "fp16"},
        # The largest: a training step of 2048 tokens.
        {"name": "glu_train_m2048_17408x5120", "kind": "glu_train", "M": 2048, "N": 17408,
         "K": 5120, "gs": 64, "bits": 4, "act": "silu", "dtype": "bf16"},
        # The down projection in a training step of 1024 tokens.
        {"name": "qmm_train_m1024_5120x17408", "kind": "qmm_train", "M": 1024, "N": 5120,
         "K": 17408, "gs": 64, "bits": 4, "dtype": "bf16"},
        # An 8-bit head over the answer's 77 tokens.
        {"name": "qmm_train_m77_65536x2048_b8", "kind": "qmm_train", "M": 77, "N": 65536,
         "K": 2048, "gs": 64, "bits": 8, "dtype": "bf16"},
        # One decoded token over the largest vocabulary of the 27B-class models.
        {"name": "sample_r1_v248320", "kind": "sample", "R": 1, "V": 248320, "dtype": "bf16",
         "mask": 0.0, "mix": "usual"},
        # A small vocabulary, temperature alone, float logits.
        {"name": "sample_r1_v32000_fp32", "kind": "sample", "R": 1, "V": 32000, "dtype": "fp32",
         "mask": 0.0, "mix": "temperature"},
        # Eight verified positions under a grammar that leaves a tenth, odd vocabulary.
        {"name": "sample_r8_v50257_fp16", "kind": "sample", "R": 8, "V": 50257, "dtype": "fp16",
         "mask": 0.9, "mix": "all"},
        # A decode batch of 64 sequences, each with settings of its own.
        {"name": "sample_r64_v248320", "kind": "sample", "R": 64, "V": 248320, "dtype": "bf16",
         "mask": 0.0, "mix": "all"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: every size log-uniform, K in whole groups, rows, columns
    and vocabularies any."""
    kind = rng.choice(["glu", "glu", "glu_train", "qmm_train", "sample", "sample"])
    if kind == "sample":
        V = _log(rng, 8000, 248320)
        return {"kind": kind, "R": _log(rng, 1, 64), "V": V, "dtype": rng.choice(["bf16", "fp16", "fp32"]),
                "mask": rng.choice([0.0, 0.0, 0.5, 0.99]),
                "mix": rng.choice(["usual", "temperature", "all"])}
    gs = rng.choice([32, 64, 64, 128])
    c = {"kind": kind, "K": max(64, gs) * _log(rng, 512 // max(64, gs), 8192 // max(64, gs)),
         "N": _log(rng, 512, 17408), "gs": gs, "bits": rng.choice([4, 4, 8]),
         "dtype": rng.choice(["bf16", "bf16", "fp16"])}
    if kind != "qmm_train":
        c["act"] = rng.choice(["silu", "silu", "gelu_tanh"])
    most = 2048 * min(1.0, 17408 * 5120 / (c["N"] * c["K"]))
    c["M"] = _log(rng, 1 if kind == "glu" else 16, most)
    return c


# ---- inputs -----------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _bank(g, c):
    """An N(0, 0.02) matrix as an affine checkpoint holds it: (uint32 words,
    scales, biases)."""
    N, K, gs, bits, dt = c["N"], c["K"], c["gs"], c["bits"], _DTYPES[c["dtype"]]
    words = torch.empty((N, K * bits // 8), dtype=torch.uint8, device="cuda")
    s = torch.empty((N, K // gs), dtype=dt, device="cuda")
    b = torch.empty_like(s)
    step = max(1, (1 << 27) // K)
    for r in range(0, N, step):
        n = min(step, N - r)
        w = torch.randn((n, K // gs, gs), generator=g, device="cuda").mul_(0.02)
        lo, hi = w.aminmax(dim=-1)
        sc = ((hi - lo) / (2 ** bits - 1)).clamp_min(1e-7).to(dt)
        bi = lo.to(dt)
        q = ((w - bi.float().unsqueeze(-1)) / sc.float().unsqueeze(-1)).round_()
        q = q.clamp_(0, 2 ** bits - 1).to(torch.uint8).reshape(n, K)
        words[r:r + n] = q if bits == 8 else q[:, 0::2] | (q[:, 1::2] << 4)
        s[r:r + n] = sc
        b[r:r + n] = bi
    return words.view(torch.int32).view(torch.uint32), s, b


def _settings(g, c):
    """Each row's temperature, top_k, top_p and min_p, and its uniform number."""
    R, cu = c["R"], "cuda"
    u = torch.rand(R, generator=g, device=cu)
    t = torch.rand(R, generator=g, device=cu) * 0.9 + 0.4
    k = torch.zeros(R, dtype=torch.int32, device=cu)
    p, m = torch.ones(R, device=cu), torch.zeros(R, device=cu)
    if c["mix"] == "usual":
        k, p = k + 40, p * 0.95
    if c["mix"] == "all":
        def some(share):
            return torch.rand(R, generator=g, device=cu) < share
        k = torch.where(some(0.6), torch.randint(1, 200, (R,), generator=g, device=cu), 0).int()
        p = torch.where(some(0.6), torch.rand(R, generator=g, device=cu) * 0.5 + 0.5, p)
        m = torch.where(some(0.4), torch.rand(R, generator=g, device=cu) * 0.1, m)
        t = torch.where(some(0.15), 0.0, t)
    return u, t, k, p, m


def prepare(case, seed):
    """What a program holds before the call: the layer's weights and the step's
    activations, or the logits and the sequences' settings."""
    c, g = case, _gen(seed)
    dt = _DTYPES[c["dtype"]]
    state = {"kind": c["kind"]}
    if c["kind"] == "sample":
        # most of a vocabulary is a bulk, a few hundred words fit, fewer well
        l = torch.randn((c["R"], c["V"]), generator=g, device="cuda").mul_(2.2)
        fit = torch.rand((c["R"], c["V"]), generator=g, device="cuda")
        l += 6.0 * (fit < 300.0 / c["V"])
        l += 4.0 * (fit < 12.0 / c["V"])
        if c["mask"]:
            out = torch.rand((c["R"], c["V"]), generator=g, device="cuda") < c["mask"]
            l = l.masked_fill(out, -math.inf)
        state["logits"] = l.to(dt)
        state["settings"] = _settings(g, c)
        return state
    state.update(gs=c["gs"], bits=c["bits"], banks=[_bank(g, c)])
    state["x"] = torch.randn((c["M"], c["K"]), generator=g, device="cuda").to(dt)
    if c["kind"] != "qmm_train":
        state["banks"].append(_bank(g, c))
        state["act"] = c["act"]
    if c["kind"] != "glu":
        state["d"] = torch.randn((c["M"], c["N"]), generator=g, device="cuda").to(dt)
    return state


# ---- one pass ---------------------------------------------------------------

def _unpack(w, bits):
    """uint32 words -> codes."""
    b = w.view(torch.uint8)
    if bits == 8:
        return b
    return torch.stack([b & 15, b >> 4], dim=-1).reshape(*b.shape[:-1], -1)


def _weight(bank, gs, bits):
    """The weights that a bank's codes stand for: rounded to T, in float32."""
    w, s, b = bank
    q = _unpack(w, bits).float().reshape(*s.shape, gs)
    v = s.float().unsqueeze(-1) * q + b.float().unsqueeze(-1)
    return v.to(s.dtype).float().reshape(w.shape[0], -1)


_TANH = math.sqrt(2 / math.pi)


def _act(g, act):
    """The activation and its derivative."""
    if act == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    # 0.5 g (1 + tanh(z)) = g / (1 + exp(-2 z)), z = sqrt(2 / pi) (g + 0.044715 g^3)
    s = 1 / (1 + torch.exp(-2 * _TANH * (g + 0.044715 * g * g * g)))
    return g * s, s + g * s * (1 - s) * 2 * _TANH * (1 + 3 * 0.044715 * g * g)


def _plain_sample(logits, u, t, k, p, m):
    l = logits.double()
    l = torch.where(torch.isnan(l), -math.inf, l)
    V = l.shape[-1]
    greedy = t <= 0
    w = torch.exp((l - l.amax(-1, keepdim=True))
                  / torch.where(greedy, 1.0, t).double().unsqueeze(-1))
    # in the order of their probability, ties to the lowest index
    ws, order = torch.sort(l, dim=-1, descending=True, stable=True)
    ws = w.gather(-1, order)
    rank = torch.arange(V, device=l.device)
    kept = rank < torch.where(k > 0, k, V).unsqueeze(-1)
    ws = torch.where(kept, ws, 0.0)
    before = torch.cumsum(ws, -1) - ws
    all_p = (p >= 1).unsqueeze(-1)
    kept &= all_p | (before < p.double().unsqueeze(-1) * ws.sum(-1, keepdim=True)) | (rank == 0)
    kept &= (ws >= m.double().unsqueeze(-1)) | (rank == 0)
    kept &= ~greedy.unsqueeze(-1) | (rank == 0)
    w = torch.zeros_like(w).scatter_(-1, order, torch.where(kept, ws, 0.0))
    # the first word whose cumulated mass is beyond u's share, in the vocabulary's order
    c = torch.cumsum(w, -1)
    token = (c > u.double().unsqueeze(-1) * c[:, -1:]).to(torch.uint8).argmax(-1)
    lp = torch.log(w.gather(-1, token.unsqueeze(-1)).squeeze(-1) / c[:, -1])
    return token.int(), lp.float()


def run(state):
    """One call or step, or its plain form."""
    kind = state["kind"]
    if kind == "sample":
        if own:
            import mlxturbo_amd as mq
            u, t, k, p, m = state["settings"]
            return mq.sample(state["logits"], u, temperature=t, top_k=k, top_p=p, min_p=m)
        return _plain_sample(state["logits"], *state["settings"])
    x, banks, gs, bits = state["x"], state["banks"], state["gs"], state["bits"]
    if own:
        import mlxturbo_amd as mq
        if kind == "glu":
            return mq.quantized_glu(x, *banks, activation=state["act"], group_size=gs, bits=bits)
        x = x.detach().requires_grad_()
        if kind == "glu_train":
            y = mq.quantized_glu(x, *banks, activation=state["act"], group_size=gs, bits=bits)
        else:
            y = mq.quantized_matmul(x, *banks[0], group_size=gs, bits=bits)
        return y.detach(), torch.autograd.grad(y, x, state["d"])[0]
    xf, ws = x.float(), [_weight(b, gs, bits) for b in banks]
    if kind == "qmm_train":
        return (torch.matmul(xf, ws[0].T).to(x.dtype),
                torch.matmul(state["d"].float(), ws[0]).to(x.dtype))
    g, v = torch.matmul(xf, ws[0].T), torch.matmul(xf, ws[1].T)
    a, da = _act(g, state["act"])
    h = (a * v).to(x.dtype)
    if kind == "glu":
        return h
    d = state["d"].float()
    return h, (torch.matmul(d * v * da, ws[0]) + torch.matmul(d * a, ws[1])).to(x.dtype)


# ---- what a pass needs ------------------------------------------------------

def work(case):
    c = case
    size = 4 if c["dtype"] == "fp32" else 2
    if c["kind"] == "sample":
        # each word's exponential, and its part in the sums
        return {"bytes": c["R"] * (c["V"] * size + 28), "flops": 4 * c["R"] * c["V"]}
    M, N, K = c["M"], c["N"], c["K"]
    bank = N * K * c["bits"] / 8 + 4 * N * K / c["gs"]
    banks = 1 if c["kind"] == "qmm_train" else 2
    train = c["kind"] != "glu"
    return {"bytes": banks * bank + 2 * (M * K + M * N) * (2 if train else 1),
            "flops": 2 * banks * M * N * K * (2 if train else 1)}


# ---- the same in 64 bits ----------------------------------------------------

def _weight64(bank, r, n, gs, bits):
    """Rows r .. r + n - 1: scale * code + bias is exact in 64 bits but for its
    last places; the float32 sum is what is rounded to T."""
    w, s, b = (t[r:r + n] for t in (bank[0].view(torch.int32), bank[1], bank[2]))
    per = 32 // bits
    sh = torch.arange(per, device=w.device) * bits
    q = ((w.long().unsqueeze(-1) >> sh) & (2 ** bits - 1)).reshape(n, -1).double()
    sb = [t.double().repeat_interleave(gs, dim=1) for t in (s, b)]
    return (sb[0] * q + sb[1]).float().to(s.dtype).double()


def _exact_train(d, act):
    x = d["x"].double()
    dy = d["d"].double() if "d" in d else None
    N, K = d["banks"][0][1].shape[0], x.shape[1]
    step = max(1, (1 << 26) // K)
    ys, dx = [], torch.zeros_like(x)
    for r in range(0, N, step):
        n = min(step, N - r)
        ws = [_weight64(b, r, n, d["gs"], d["bits"]) for b in d["banks"]]
        y = [x @ w.T for w in ws]
        if act is None:
            ys.append(y[0])
            dx += dy[:, r:r + n] @ ws[0]
            continue
        g, v = y
        if act == "silu":
            s = torch.sigmoid(g)
            a, da = g * s, s + g * s * (1 - s)
        else:
            c = math.sqrt(2 / math.pi)
            th = torch.tanh(c * (g + 0.044715 * g ** 3))
            a = 0.5 * g * (1 + th)
            da = 0.5 * (1 + th) + 0.5 * g * (1 - th * th) * c * (1 + 3 * 0.044715 * g * g)
        ys.append(a * v)
        if dy is not None:
            e = dy[:, r:r + n]
            dx += (e * v * da) @ ws[0] + (e * a) @ ws[1]
    return torch.cat(ys, dim=-1), dx


def _exact_row(l, u, t, k, p, m):
    """One row's token and its log probability, from numpy's float64 values."""
    import numpy as np
    l = np.where(np.isnan(l), -np.inf, l)
    order = np.lexsort((np.arange(l.size), -l))
    if t <= 0:
        return int(order[0]), 0.0
    w = np.exp((l - l[order[0]]) / t)
    n = min(k, l.size) if k > 0 else l.size
    top = w[order[:n]]
    if p < 1:
        cum = np.cumsum(top)
        n = max(1, int(np.searchsorted(cum, p * cum[-1], side="left")) + 1)
        top = top[:n]
    n = max(1, int(np.count_nonzero(top >= m)))
    ids = np.sort(order[:n])
    cum = np.cumsum(w[ids])
    i = int(ids[min(int(np.searchsorted(cum, u * cum[-1], side="right")), n - 1)])
    return i, float(np.log(w[i]) - np.log(cum[-1]))


def exact(case, seed):
    """`run` on the same inputs in float64."""
    d = prepare(case, seed)
    if case["kind"] == "sample":
        rows = [_exact_row(l, *row) for l, *row in zip(
            d["logits"].double().cpu().numpy(), *(s.double().tolist() if i != 2 else s.tolist()
                                                  for i, s in enumerate(d["settings"])))]
        return (torch.tensor([r[0] for r in rows], dtype=torch.int32),
                torch.tensor([r[1] for r in rows], dtype=torch.float64))
    y, dx = _exact_train(d, case.get("act"))
    return y if case["kind"] == "glu" else (y, dx)
