"""Accumulated attention weights and eviction by them (oracle; test infrastructure only).

``weights`` is the softmax of ``window.attend`` summed over queries and the query heads of a KV head (float64); pinned in
tests/test_oracle_evict.py by its total (queries x heads). ``evict`` works on plain lists from the rule alone; pinned there by
hand-written cases and by what a full sort keeps.
"""
from __future__ import annotations

import math

import numpy as np

from . import window as ow


def weights(q, k, v, q_pos, scale: float) -> np.ndarray:
    """float64 [8, m]: what the queries q [n, 32, D] at positions q_pos give the rows k [m, 8, D] (causal)."""
    m = k.shape[0]
    w = ow.attend(q, k, v, ow.visible(q_pos, m, m + max(q_pos) + 1, 0), scale)[2]
    return w.reshape(k.shape[1], -1, w.shape[1], m).sum((1, 2))


def evict(scores, positions, tokens: int, budget: int, sinks: int, recent: int):
    """One (layer, sequence, head): scores and positions of its n rows. Returns (moves [(from, to)], scores, positions), the
    latter as they are afterwards; None for a sequence within its budget."""
    n = len(scores)
    m = min(n, budget)
    if n <= m:
        return None
    pos = [tokens - (n - s) if p < 0 else int(p) for s, p in enumerate(positions)]
    held = [p < sinks or p >= tokens - recent for p in pos]

    def rank(s):
        x = float(scores[s])
        return (0 if held[s] else 1, 0 if not math.isnan(x) else 1, -x if not math.isnan(x) and not held[s] else 0, s)

    kept = set(sorted(range(n), key=rank)[:m])
    holes = [s for s in range(m) if s not in kept]
    movers = [s for s in range(m, n) if s in kept]
    moves = list(zip(movers, holes))
    new_s, new_p = np.array(scores, np.float32), np.array(positions, np.int32)
    for s in kept:
        if s < m:
            new_p[s] = pos[s]
    for src, dst in moves:
        new_s[dst], new_p[dst] = scores[src], pos[src]
    new_s[m:], new_p[m:] = 0, -1
    return moves, new_s, new_p
