"""The oracle of the paged operators against closed forms (no device)."""

import math

import numpy as np

import paged_oracle as po


def test_plan_gives_out_and_takes_back():
    table = [[4, 5, -1], [0, -1, -1], [7, 3, -1]]
    got = po.plan([30, 16, 20], [3, -1, 1], [2, 1, 2], 16, table, [9, 8, 6, -1, -1, -1, -1, -1, -1, -1], 3, 8)
    # page 0 comes back on top; request 0 needs a third page and takes it
    assert got["served"] == 3 and got["err"] == 0 and got["count"] == 3
    assert got["table"].tolist() == [[4, 5, 0], [0, -1, -1], [7, 3, -1]]
    assert got["free"][:4].tolist() == [9, 8, 6, 0]
    assert got["cu"].tolist() == [0, 3, 3, 4] and got["lengths"].tolist() == [33, 0, 21] and got["held"].tolist() == [3, 0, 2]
    assert got["slot"][:4].tolist() == [5 * 16 + 14, 5 * 16 + 15, 0, 3 * 16 + 4]
    assert got["position"].tolist() == [30, 31, 32, 20, -1, -1, -1, -1]


def test_plan_stops_at_the_first_that_does_not_fit():
    got = po.plan([16, 16, 0, 5], [1, 1, 0, 1], [1, 1, 0, 1], 16, [[0, -1], [1, -1], [-1, -1], [2, -1]], [3, -1, -1, -1], 1, 8)
    assert got["served"] == 1 and got["cu"].tolist() == [0, 1, 1, 1, 1] and got["count"] == 0
    assert got["lengths"].tolist() == [17, 16, 0, 5]


def test_attention_of_equal_scores_is_a_mean():
    rng = np.random.default_rng(1)
    k, v = rng.standard_normal((2, 9, 1, 8))
    out, bound = po.attention(np.zeros((2, 2, 8)), k, v, 9, window=4, sinks=2)
    assert np.allclose(out[0, 1], v[[0, 1, 4, 5, 6, 7], 0].mean(axis=0)) and np.allclose(out[1, 0], v[[0, 1, 5, 6, 7, 8], 0].mean(axis=0))
    assert (bound > 0).all() and bound.max() < 1e-4
    empty, _ = po.attention(np.ones((3, 2, 8)), k[:1], v[:1], 1)
    assert not empty[:2].any() and np.allclose(empty[2], v[0, 0])


def test_verification_by_hand():
    p, q = np.log(np.float32([0.5, 0.25, 0.25])), np.log(np.float32([0.25, 0.5, 0.25]))
    one = (1.0, 0, 1.0, 0.0)
    # id 0: q < p, accepted whatever u; id 1: accepted below 0.5; after a rejection max(p - q, 0) is id 0 alone
    assert po.verify([p, p], [0], [q], one, [0.99], 0.6) == ([0, 1], 1)
    assert po.verify([p, p], [1], [q], one, [0.49], 0.8) == ([1, 2], 1)
    assert po.verify([p, p], [1], [q], one, [0.51], 0.99) == ([0, -1], 0)
    # looked up: accepted below p, then p without it
    assert po.verify([p, p], [0], None, one, [0.4], 0.0) == ([0, 0], 1)
    assert po.verify([p, p], [0], None, one, [0.6], 0.51) == ([2, -1], 0)
    # every id comes out with probability p, whatever q is
    count = np.zeros(3)
    n = 24
    for t, w in ((0, 0.25), (1, 0.5), (2, 0.25)):
        for u in (np.arange(n) + 0.5) / n:
            for d in (np.arange(n) + 0.5) / n:
                count[po.verify([p, p], [t], [q], one, [u], d)[0][0]] += w / n / n
    assert np.abs(count - [0.5, 0.25, 0.25]).max() < 1 / n


def test_masses_keep_what_the_settings_say():
    logits = np.float32([2, 1, 3, 1, -np.inf, np.nan])
    m, total = po.masses(logits, 1.0, 0, 1.0, 0.0)
    assert np.allclose(m[:4] / total, np.exp([-1, -2, 0, -2]) / np.exp([-1, -2, 0, -2]).sum()) and not m[4:].any()
    assert (po.masses(logits, 1.0, 3, 1.0, 0.0)[0] > 0).tolist() == [True, True, True, False, False, False]
    assert po.masses(logits, 0.0, 0, 1.0, 0.0)[0].tolist() == [0, 0, 1, 0, 0, 0]
    assert (po.masses(logits, 1.0, 0, 0.7, 0.0)[0] > 0).sum() == 2 and math.isclose(po.masses(logits, 1.0, 0, 1.0, 0.3)[1], 2.0 ** 44 * (1 + math.exp(-1)), rel_tol=1e-9)
