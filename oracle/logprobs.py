"""Log probabilities, entropy, alternatives and their gradient (oracle; test infrastructure only): float64 from the definition,
checked by central differences in tests/test_oracle_logprobs.py."""
from __future__ import annotations

import numpy as np


def forward(logits, targets, temperature=1.0):
    """logits [T, V] float64: log softmax [T, V], the targets' log probabilities (0 outside [0, V)), entropies."""
    x = logits / temperature
    with np.errstate(all="ignore"):
        m = x.max(1, keepdims=True)
        ls = x - m - np.log(np.exp(x - m).sum(1, keepdims=True))
        p = np.exp(ls)
        ent = -np.where(p > 0, p * ls, 0).sum(1) + np.where(np.isnan(ls[:, 0]), np.nan, 0)
    rows = np.arange(len(x))
    real = (targets >= 0) & (targets < x.shape[1])
    lp = np.where(real, ls[rows, np.where(real, targets, 0)], 0.0)
    return ls, lp, ent


def top(logits, n):
    """Ids of the n highest logits, ties by the lower id, NaN as -inf."""
    return np.argsort(-np.where(np.isnan(logits), -np.inf, logits), axis=1, kind="stable")[:, :n]


def backward(logits, targets, dlogp, dent, temperature=1.0):
    """Gradient of sum(dlogp logp + dent H)."""
    ls, _, ent = forward(logits, targets, temperature)
    p = np.exp(ls)
    real = (targets >= 0) & (targets < logits.shape[1])
    g = np.where(real, dlogp, 0.0)
    with np.errstate(all="ignore"):
        d = np.where(p > 0, -p * (g[:, None] + dent[:, None] * (ls + ent[:, None])), 0.0)
    d[np.arange(len(d))[real], targets[real]] += g[real]
    return d / temperature
