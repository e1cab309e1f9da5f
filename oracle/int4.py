"""Cache rows in 4 bits and attention over them (oracle; test infrastructure only).

Rows are quantised and read in numpy from the format's definition, dim by dim; attention is float64 over the values that the rows
stand for. Its bounds say how far a kernel may be off: it takes a weight times its row's step, in two bf16 parts (half a step
of the second, 2^-16 of it), against 128 + code and -136 in fp32 sums, and the weight in fp32 against the group's middle, and rounds
the output; split partials are fp16 (2^-11 of the split's largest output, itself at most the largest value; ``whole``: none). ``wide``: the multi-query kernel instead takes
values and weights in fp16 (half a step, 2^-11 of each; its powers of two keep them, and what is 2^-19 of its row's or page's largest,
in the type's normal range; weights down to 2^-25 of the row's largest, and what lies below is off by up to 2^-36 of that, which is
not in the bounds), and its partials are fp32.
"""
from __future__ import annotations

import numpy as np

HEADS, DIM, GROUP = 8, 128, 32
EPS = 2.0 ** -8
HALF = 2.0 ** -11              # of fp16
SLACK = 1.02


def bf16(x):
    """float32 values rounded to bf16 (nearest even), as float32."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)
    return np.where(np.isnan(x), np.float32(np.nan), r)


def place(d: int) -> tuple[int, int]:
    """(word of the head's 16, first bit) of dim d."""
    b = d // 8
    return 4 * (b % 4) + b // 4, 4 * (d % 8 // 2) + 16 * (d % 2)


def quantise(x: np.ndarray) -> np.ndarray:
    """bf16 rows [n, 8, 128] (as float32) -> bytes [n, 640]."""
    n = len(x)
    words = np.zeros((n, HEADS, 16), np.uint32)
    pairs = np.zeros((n, HEADS, 4, 2), np.float32)
    with np.errstate(all="ignore"):
        for g in range(4):
            v = x[:, :, GROUP * g: GROUP * (g + 1)].astype(np.float32)
            lo, hi = v.min(-1), v.max(-1)
            span = hi - lo
            good = np.isfinite(v).all(-1) & np.isfinite(span)
            step = np.where(good, bf16(span / np.float32(15)), np.float32(np.nan))
            pairs[:, :, g, 0], pairs[:, :, g, 1] = step, np.where(good, lo, 0)
            code = np.minimum(np.rint((v - lo[..., None]) / step[..., None]), 15)
            code = np.where((step > 0)[..., None], code, 0).astype(np.uint32)
            for i in range(GROUP):
                w, bit = place(GROUP * g + i)
                words[:, :, w] |= code[:, :, i] << np.uint32(bit)
    raw = (pairs.view(np.uint32) >> 16).astype(np.uint16)
    raw[np.isnan(pairs)] = 0x7FC0
    return np.concatenate([words.reshape(n, 128).view(np.uint8), raw.reshape(n, 64).view(np.uint8)], 1)


def split(rows: np.ndarray):
    """Bytes [n, 640] -> steps and minima [n, 8, 4] and codes [n, 8, 128], float64."""
    n = len(rows)
    words = np.ascontiguousarray(rows[:, :512]).view(np.uint32).reshape(n, HEADS, 16)
    pairs = (np.ascontiguousarray(rows[:, 512:]).view(np.uint16).astype(np.uint32) << 16).view(np.float32)
    pairs = pairs.reshape(n, HEADS, 4, 2).astype(np.float64)
    codes = np.empty((n, HEADS, DIM))
    for d in range(DIM):
        w, bit = place(d)
        codes[:, :, d] = (words[:, :, w] >> np.uint32(bit)) & 15
    return pairs[..., 0], pairs[..., 1], codes


def values(rows: np.ndarray) -> np.ndarray:
    """Bytes [n, 640] -> float64 [n, 8, 128]."""
    step, lo, codes = split(rows)
    return np.repeat(lo, GROUP, -1) + np.repeat(step, GROUP, -1) * codes


def attend(q, k_rows, v_rows, vis, scale: float, wide: bool = False, whole: bool = False):
    """q [n, 32, 128] float64 over m rows of bytes, vis [n, m]: out [n, 32, 128], lse [n, 32] and the bounds of both (rows that
    see nothing: 0 and -inf)."""
    n = len(q)
    ks, _, _ = split(k_rows)
    k, v = values(k_rows), values(v_rows)
    vs, vlo, vc = split(v_rows)
    part = np.repeat(vs, GROUP, -1) * np.abs(vc - 8)                     # what a rounded weight multiplies
    mid = np.abs(np.repeat(vlo + 8 * vs, GROUP, -1))
    summed = 143 * np.repeat(vs, GROUP, -1) + mid                        # what the sums hold, 32 rows at a time, a step after another
    adds = (len(v) / 32 + 40) * 2.0 ** -24
    out, lse = np.zeros((n, 32, DIM)), np.full((n, 32), -np.inf)
    tol, ltol = np.zeros_like(out), np.zeros((n, 32))
    some = vis.any(1)
    for h in range(32):
        u = h // 4
        s = np.where(vis, (q[:, h] @ k[:, u].T) * scale, -np.inf)[some]
        if s.size == 0:
            continue
        # Scores in fp32: sums of up to 40 products (8 a lane, 4 lanes, the start of -128 sum q) of |q| (128 + c) s, beside the
        # minimum's part; wide: of values rounded to fp16, in sums of 128
        size = np.abs(q[some, h]) @ (np.abs(k[:, u]) + (0 if wide else 136 * np.repeat(ks[:, u], GROUP, -1))).T
        ds = scale * size * (128 * 2.0 ** -24 + HALF if wide else 40 * 2.0 ** -24) + 2.0 ** -22 * np.abs(np.where(vis[some], s, 0))
        ds = np.where(vis[some], ds, 0)
        m = s.max(1, keepdims=True)
        p = np.exp(s - m)
        z = p.sum(1, keepdims=True)
        w = p / z
        lse[some, h] = (m + np.log(z))[:, 0]
        o = w @ v[:, u]
        out[some, h] = o
        # a score off by ds moves the output by w ds (v - out), twice that for the sum's own
        moved = (w * ds) @ np.abs(v[:, u]) + (w * ds).sum(1, keepdims=True) * np.abs(o)
        err = HALF * (w @ (2 * np.abs(v[:, u]))) if wide else EPS ** 2 * (w @ part[:, u]) + adds * (w @ summed[:, u])
        floor = 2.0 ** -20 if wide or whole else 2.0 ** -11
        tol[some, h] = SLACK * (err + moved + EPS * np.abs(o)) + floor * np.abs(v[:, u]).max(initial=0)
        ltol[some, h] = ds.max(1) + (HALF if wide else 0) + 1e-5
    return out, lse, tol, ltol
