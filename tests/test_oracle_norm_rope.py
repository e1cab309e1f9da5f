"""The norm-and-rotation oracle: closed forms, and its gradients by central differences."""
import numpy as np

from oracle import norm_rope as on

RNG = np.random.default_rng(0)


def test_closed_forms():
    x, w = RNG.standard_normal((5, 128)), RNG.standard_normal(128)
    one, none = np.ones((5, 64)), np.zeros((5, 64))
    y = on.forward(x, w, one, none, 0.0)                     # no rotation: the norm alone
    assert np.allclose((y / w) ** 2 @ np.ones(128), 128)
    quarter = on.forward(x, w, none, one, 0.0)
    assert np.allclose(quarter, np.concatenate([-y[:, 64:], y[:, :64]], 1))
    a = RNG.standard_normal((5, 64))
    assert np.allclose(on.rotate(on.rotate(x, np.cos(a), np.sin(a)), np.cos(a), -np.sin(a)), x)
    assert np.allclose(on.forward(np.zeros((1, 128)), w, one[:1], none[:1], 1e-6), 0)


def test_gradients_by_differences():
    x, w, a = RNG.standard_normal((3, 128)), 1 + 0.3 * RNG.standard_normal(128), RNG.standard_normal((3, 64))
    c, s, dout = np.cos(a), np.sin(a), RNG.standard_normal((3, 128))
    dx, dw = on.backward(x, w, c, s, 1e-3, dout)
    f = lambda x, w: (dout * on.forward(x, w, c, s, 1e-3)).sum()             # noqa: E731
    h = 1e-6
    for i in range(3):
        for d in range(0, 128, 11):
            e = np.zeros_like(x)
            e[i, d] = h
            assert abs((f(x + e, w) - f(x - e, w)) / (2 * h) - dx[i, d]) < 1e-7
    for d in range(0, 128, 11):
        e = np.zeros_like(w)
        e[d] = h
        assert abs((f(x, w + e) - f(x, w - e)) / (2 * h) - dw[d]) < 1e-7
