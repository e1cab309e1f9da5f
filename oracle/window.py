"""Attention under a sliding window with sinks (oracle; test infrastructure only).

float64, from the definition: row i sees key j when j <= i and (i - j < window or j < sinks). ``attend`` is pinned by
closed forms and by ``decode.decode_fp64`` in tests/test_oracle_window.py, the gradients by central differences there.

``bounds=True`` adds, per output element, how far a bf16 kernel may be off by arithmetic alone. With e = 2^-8 (half a step
of bf16, relative) and weights w, such a kernel rounds each weight before the product with v and divides by the sum of the
rounded weights, |err| <= e (sum w |v| + |out|), then rounds the output, e |out|. Backwards it takes lse from the rounded sum
(each P off by e), rounds P and dS (e each), takes D from the rounded output, and rounds the result. SLACK covers the second
order and the fp32 sums.
"""
from __future__ import annotations

import numpy as np

EPS = 2.0 ** -8
SLACK = 1.02
FP32 = 2e-5                     # scores of |q . k| <= ~50 in fp32, relative error of a weight


def visible(q_pos, n_keys: int, window: int, sinks: int) -> np.ndarray:
    """bool [len(q_pos), n_keys]."""
    i, j = np.asarray(q_pos)[:, None], np.arange(n_keys)[None, :]
    return (j <= i) & ((i - j < window) | (j < sinks))


def attend(q, k, v, vis, scale: float, bounds: bool = False):
    """q [n, 32, D], k, v [m, 8, D] float64, vis [n, m]: out [n, 32, D], lse [n, 32], weights [32, n, m] (rows that see
    nothing: 0, -inf, 0); with ``bounds`` also the bound of out."""
    n, H, D = q.shape
    G = H // k.shape[1]
    out, lse, w = np.zeros((n, H, D)), np.full((n, H), -np.inf), np.zeros((H, n, k.shape[0]))
    tol = np.zeros_like(out)
    some = vis.any(1)
    for h in range(H):
        s = np.where(vis, (q[:, h] @ k[:, h // G].T) * scale, -np.inf)[some]
        if s.size == 0:
            continue
        m = s.max(1, keepdims=True)
        p = np.exp(s - m)
        z = p.sum(1, keepdims=True)
        w[h, some] = p / z
        lse[some, h] = (m + np.log(z))[:, 0]
        out[:, h] = w[h] @ v[:, h // G]
        if bounds:
            tol[:, h] = SLACK * EPS * (w[h] @ np.abs(v[:, h // G]) + 2 * np.abs(out[:, h])) + FP32 * (
                w[h] @ np.abs(v[:, h // G]))
    return (out, lse, w, tol) if bounds else (out, lse, w)


def window_attention(q, k, v, lens, window: int, sinks: int, scale: float, bounds: bool = False):
    """Whole prompts [B, S, heads, D]: out [B, S, 32, D], lse [B, 32, S] and, with ``bounds``, the bound of out."""
    B, S = q.shape[:2]
    out, lse, tol = np.zeros(q.shape), np.full((B, q.shape[2], S), -np.inf), np.zeros(q.shape)
    for b in range(B):
        n = S if lens is None else int(lens[b])
        if n == 0:
            continue
        vis = visible(np.arange(n), n, window, sinks)
        got = attend(q[b, :n], k[b, :n], v[b, :n], vis, scale, bounds)
        out[b, :n], lse[b, :, :n] = got[0], got[1].T
        if bounds:
            tol[b, :n] = got[3]
    return (out, lse, tol) if bounds else (out, lse)


def window_backward(q, k, v, dout, lens, window: int, sinks: int, scale: float, bounds: bool = False):
    """dq, dk, dv of sum(dout * out); with ``bounds`` a bound per element after each."""
    B, S, H, D = q.shape
    G = H // k.shape[2]
    grads = [np.zeros(t.shape) for t in (q, k, v)]
    tols = [np.zeros(t.shape) for t in (q, k, v)]
    for b in range(B):
        n = S if lens is None else int(lens[b])
        if n == 0:
            continue
        vis = visible(np.arange(n), n, window, sinks)
        out, _, w, otol = attend(q[b, :n], k[b, :n], v[b, :n], vis, scale, True)
        for h in range(H):
            qh, kh, vh, g, p = q[b, :n, h], k[b, :n, h // G], v[b, :n, h // G], dout[b, :n, h], w[h]
            dp, d = g @ vh.T, (g * out[:, h]).sum(1, keepdims=True)
            ds = p * (dp - d)
            grads[0][b, :n, h] = scale * ds @ kh
            grads[1][b, :n, h // G] += scale * ds.T @ qh
            grads[2][b, :n, h // G] += p.T @ g
            if bounds:
                dtol = (np.abs(g) * otol[:, h]).sum(1, keepdims=True) + FP32 * np.abs(g).max() * np.abs(vh).max() * 11.4
                err = p * dtol + 2 * EPS * np.abs(ds) + FP32 * p * (np.abs(dp) + np.abs(d))
                tols[0][b, :n, h] = scale * err @ np.abs(kh)
                tols[1][b, :n, h // G] += scale * err.T @ np.abs(qh)
                tols[2][b, :n, h // G] += (2 * EPS + FP32) * p.T @ np.abs(g)
    if not bounds:
        return tuple(grads)
    return tuple(x for g, t in zip(grads, tols) for x in (g, SLACK * (t + EPS * np.abs(g))))
