"""The log-probability oracle: scipy, closed forms, differences."""
import numpy as np
from scipy.special import log_softmax
from scipy.stats import entropy

from oracle import logprobs as ol

RNG = np.random.default_rng(0)


def test_closed_forms():
    x, t = RNG.standard_normal((6, 40)) * 3, RNG.integers(0, 40, 6)
    t[2] = -100
    ls, lp, ent = ol.forward(x, t, 0.7)
    want = log_softmax(x / 0.7, 1)
    assert np.allclose(ls, want) and lp[2] == 0 and np.allclose(lp[0], want[0, t[0]])
    assert np.allclose(ent, entropy(np.exp(want), axis=1))
    x[1, 3:] = -np.inf
    assert abs(ol.forward(np.zeros((1, 8)), t[:1] % 8)[2][0] - np.log(8)) < 1e-12
    assert np.isfinite(ol.forward(x, t)[2]).all()
    assert ol.top(np.array([[1.0, 3.0, np.nan, 3.0, -np.inf]]), 5).tolist() == [[1, 3, 0, 2, 4]]


def test_gradient_by_differences():
    x, t = RNG.standard_normal((3, 9)), np.array([4, -1, 0])
    g, h = RNG.standard_normal(3), RNG.standard_normal(3)
    d = ol.backward(x, t, g, h, 1.3)

    def f(x):
        _, lp, ent = ol.forward(x, t, 1.3)
        return (g * lp + h * ent).sum()

    for i in range(3):
        for v in range(9):
            e = np.zeros_like(x)
            e[i, v] = 1e-6
            assert abs((f(x + e) - f(x - e)) / 2e-6 - d[i, v]) < 1e-8
