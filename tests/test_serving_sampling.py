"""When the tokens of a draft check follow the target's probabilities: the rule
of include/myl_hip.h in exact fractions, over every draft and random number."""
from __future__ import annotations

from fractions import Fraction

import numpy as np

import serving_ref as ref


def next_token(p, q, t):
    """The distribution of the first token after draft t: q the draft's weights, None without."""
    P, V = int(p.sum()), len(p)
    Q = 1 if q is None else int(q.sum())
    q = [int(j == t) for j in range(V)] if q is None else [int(x) for x in q]
    take = Fraction(1) if q[t] == 0 and p[t] else min(Fraction(1), Fraction(int(p[t]) * Q, q[t] * P)) if q[t] else Fraction(0)
    rest = [max(0, int(p[j]) * Q - q[j] * P) for j in range(V)]
    rest = rest if sum(rest) else [int(x) for x in p]
    return [take * (j == t) + (1 - take) * Fraction(rest[j], sum(rest)) for j in range(V)]


def mixed(p, q, drafts):
    """The same over drafts of these probabilities."""
    rows = [(w, next_token(p, q, t)) for t, w in enumerate(drafts) if w]
    return [sum(w * r[j] for w, r in rows) for j in range(len(p))]


def test_which_drafts_leave_the_targets_distribution():
    r = np.random.default_rng(5)
    lut = np.round(np.exp(-np.arange(2662) / 256) * 16384).astype(np.int16)
    biased = 0
    for case in range(40):
        V = int(r.integers(2, 9))
        p, q = (ref.row_weights(r.integers(-300, 300, V).astype(np.int32), lut) for _ in range(2))
        want = [Fraction(int(x), int(p.sum())) for x in p]
        # drafts drawn from the weights of the logits that are handed over
        assert mixed(p, q, [Fraction(int(x), int(q.sum())) for x in q]) == want
        # any drafts at all, handed over without probabilities
        any_drafts = [Fraction(int(x), 100) for x in r.multinomial(100, np.full(V, 1 / V))]
        assert mixed(p, None, any_drafts) == want
        assert mixed(p, None, [Fraction(int(j == q.argmax())) for j in range(V)]) == want
        # the draft's argmax handed over with its logits is taken for a sample of them
        biased += mixed(p, q, [Fraction(int(j == q.argmax())) for j in range(V)]) != want
    assert biased > 30
