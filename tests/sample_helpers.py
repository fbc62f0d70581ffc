"""Sampling from the definition, one row at a time in numpy's float64 and Python's
integers, for its tests."""

import numpy as np

INF = float("inf")


def sample_row(l, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, log probability, margin) of one row: the margin is how far, in units of
    the kept mass, u's place is from the nearest end of the token's share, and top_p's
    mass and min_p from the nearest word's; a float32 place within 2^-30 of an end may
    round either way."""
    l = np.asarray(l, np.float64)
    l = np.where(np.isnan(l), -INF, l)
    temperature = float(np.float32(temperature))
    words = np.nonzero(l > -INF)[0]
    if words.size == 0:
        return -1, -INF, INF
    order = words[np.lexsort((words, -l[words]))]
    if not temperature > 0:
        return int(order[0]), 0.0, INF
    top = l[order[0]]
    with np.errstate(invalid="ignore", over="ignore"):
        z = np.where(l == top, 0.0, (l - top) / np.float64(temperature))
    w = np.where(z > -40, np.exp(np.where(z > -40, z, 0.0)), 0.0)
    if top_p <= 0:
        top_k = 1
    n = min(top_k, order.size) if top_k > 0 else order.size
    kept = order[:n]
    margin = INF
    if 0 < top_p < 1:
        before = np.concatenate([[0.0], np.cumsum(w[kept])])
        goal = np.float64(np.float32(top_p)) * before[-1]
        # only words of mass move the cut by more than rounding
        margin = min(margin, np.abs(before[1:] - goal)[w[kept] > 0].min() / before[-1])
        kept = kept[:max(1, int(np.count_nonzero(before[:-1] < goal)))]
    if min_p > 0:
        m = np.float64(np.float32(min_p))
        margin = min(margin, np.abs(w[kept] - m).min() if m < 1 else INF)
        kept = kept[:max(1, int(np.count_nonzero(w[kept] >= m)))]
    ids = np.sort(kept)
    cum = np.cumsum(w[ids])
    t = min(max(np.float64(np.float32(u)), 0.0), 1.0) * cum[-1]
    i = int(np.searchsorted(cum, t, side="right"))
    if i >= ids.size:
        i = int(np.nonzero(w[ids])[0][-1])
    if ids.size > 1:
        margin = min(margin, np.abs(cum[:-1] - t).min() / cum[-1] if t < cum[-1] else 0.0)
    return int(ids[i]), float(z[ids[i]] - np.log(cum[-1])), margin
