"""The sampling oracle (sample_helpers.py) against the definition in whole numbers, word by
word, on random short rows (CPU)."""

import math
import random
from fractions import Fraction

import numpy as np

from sample_helpers import sample_row


def brute_force(masses, u, top_k, top_p, min_p):
    """(token, its share) of whole masses: each word is looked at by itself."""
    def before(i):
        """The words in front of word i, larger or equal ones of lower index."""
        return [j for j, m in enumerate(masses) if (m, -j) > (masses[i], -i)]

    words = [i for i, m in enumerate(masses) if m]
    first = max(words, key=lambda i: (masses[i], -i))
    if top_p <= 0:
        top_k = 1
    kept = [i for i in words if not top_k or len(before(i)) < top_k]
    if 0 < top_p < 1:
        goal = top_p * sum(masses[i] for i in kept)
        kept = [i for i in kept if sum(masses[j] for j in before(i)) < goal]
    kept = [i for i in kept if i == first or masses[i] >= min_p * masses[first]]
    total = sum(masses[i] for i in kept)
    run = 0
    for i in kept:
        run += masses[i]
        if run > u * total:
            return i, Fraction(masses[i], total)
    raise AssertionError("u is below 1")


def test_oracle_is_the_definition():
    rng = random.Random(1)
    near = 0
    for _ in range(3000):
        n = rng.randint(1, 12)
        masses = [rng.choice([0, 1, 1, 2, 3, rng.randint(1, 50)]) for _ in range(n)]
        if not any(masses):
            masses[rng.randrange(n)] = 1
        u, top_p, min_p = (float(np.float32(v)) for v in (
            rng.random() * 0.999, rng.choice([1.0, 1.0, rng.random(), 0.0]),
            rng.choice([0.0, 0.0, rng.random()])))
        top_k = rng.choice([0, 0, rng.randint(1, n + 2)])
        temperature = rng.choice([1.0, 0.5, 2.0])
        logits = [temperature * math.log(m) if m else rng.choice([-math.inf, math.nan])
                  for m in masses]
        token, logprob, margin = sample_row(logits, u, temperature, top_k, top_p, min_p)
        if margin < 1e-9:                       # logarithms are rounded
            near += 1
            continue
        want, share = brute_force(masses, Fraction(u), top_k, Fraction(top_p), Fraction(min_p))
        assert token == want, (masses, u, top_k, top_p, min_p)
        assert abs(logprob - math.log(share)) < 1e-9
    assert near < 60


def test_temperature_zero_and_ties():
    rng = random.Random(2)
    for _ in range(200):
        masses = [rng.randint(1, 3) for _ in range(rng.randint(1, 9))]
        logits = [math.log(m) for m in masses]
        assert sample_row(logits, rng.random(), 0.0)[0] == masses.index(max(masses))
        assert sample_row(logits, rng.random(), top_k=1)[0] == masses.index(max(masses))
