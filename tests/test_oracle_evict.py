"""The eviction oracle: hand-written cases, a full sort, and the total of the accumulated weights."""
import numpy as np

from oracle import evict as oe


def test_weights_total_is_queries_times_heads():
    rng = np.random.default_rng(0)
    q, k, v = (rng.standard_normal(s) for s in ((5, 32, 128), (9, 8, 128), (9, 8, 128)))
    w = oe.weights(q, k, v, np.arange(4, 9), 128 ** -0.5)
    assert w.shape == (8, 9) and np.allclose(w.sum(1), 5 * 4)
    assert (w[:, 8] > 0).all()                               # seen by the last query only
    one = oe.weights(q[:1], k[:1], v[:1], np.array([0]), 128 ** -0.5)
    assert np.allclose(one, 4)


def test_by_hand():
    # rows 0 .. 5 of tokens 0 .. 5, budget 4, one sink, one recent: rows 1 .. 4 compete for two places
    moves, s, p = oe.evict([0.0, 1.0, 5.0, 1.0, 2.0, 0.0], [-1] * 6, 6, 4, 1, 1)
    assert moves == [(4, 1), (5, 3)]
    assert s.tolist() == [0.0, 2.0, 5.0, 0.0, 0.0, 0.0] and p.tolist() == [0, 4, 2, 5, -1, -1]
    # the same rows within the budget
    assert oe.evict([0.0] * 6, [-1] * 6, 6, 6, 1, 1) is None
    # ties go to the lowest row, NaN is below every number
    moves, s, p = oe.evict([1.0, float("nan"), 1.0, 1.0, -7.0], [-1] * 5, 5, 3, 0, 0)
    assert moves == [(3, 1)] and p.tolist() == [0, 3, 2, -1, -1]
    # positions of earlier evictions: tokens 9 and 10 were appended, tokens 2, 8 are held as sink and recent row
    moves, s, p = oe.evict([0.5, 9.0, 0.1, 0.2, 0.3], [8, 4, 2, -1, -1], 11, 4, 3, 3)
    assert moves == [(4, 1)] and p.tolist() == [8, 10, 2, 9, -1]


def test_keeps_what_a_sort_keeps():
    rng = np.random.default_rng(1)
    for _ in range(50):
        n = int(rng.integers(2, 60))
        s = rng.integers(0, 9, n).astype(np.float32)
        m = int(rng.integers(1, n))
        moves, after, p = oe.evict(s, [-1] * n, n, m, 0, 0)
        best = sorted(s, reverse=True)[:m]
        assert sorted(after[:m], reverse=True) == best and len(set(p[:m].tolist())) == m
        assert all(src >= m > dst for src, dst in moves)
