"""Per-head RMS norms with the position rotation (oracle; test infrastructure only): float64, forward and gradients from the
formula; the gradients are checked by central differences in tests/test_oracle_norm_rope.py."""
from __future__ import annotations

import numpy as np


def rotate(y, c, s):
    """Rows y [..., 128] by the angles' cosines and sines [..., 64] (NeoX halves)."""
    a, b = y[..., :64], y[..., 64:]
    return np.concatenate([a * c - b * s, b * c + a * s], -1)


def forward(x, w, c, s, eps):
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    return rotate(x * r * w, c, s)


def backward(x, w, c, s, eps, dout):
    """(dx, dw) of sum(dout * forward)."""
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    dy = rotate(dout, c, -s)
    g = dy * w
    dx = r * (g - x * r * r * (g * x).mean(-1, keepdims=True))
    return dx, (dy * x * r).reshape(-1, x.shape[-1]).sum(0)
