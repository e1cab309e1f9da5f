"""The sliding-window oracle: closed forms, agreement with the decode oracle, gradients against central differences."""
import numpy as np
import pytest

from oracle import decode as od
from oracle import window as ow

SCALE = 128 ** -0.5


def _rand(rng, *shape):
    return rng.standard_normal(shape)


def test_visible_by_definition():
    for window in (1, 2, 5, 100):
        for sinks in (0, 1, 3, 50):
            vis = ow.visible(np.arange(3, 11), 12, window, sinks)
            for a, i in enumerate(range(3, 11)):
                for j in range(12):
                    assert vis[a, j] == (j <= i and (i - j < window or j < sinks))


def test_window_one_without_sinks_copies_values():
    rng = np.random.default_rng(0)
    q, k, v = _rand(rng, 1, 9, 32, 128), _rand(rng, 1, 9, 8, 128), _rand(rng, 1, 9, 8, 128)
    out, lse = ow.window_attention(q, k, v, None, 1, 0, SCALE)
    assert np.allclose(out, np.repeat(v, 4, axis=2))
    s = np.einsum("bshd,bshd->bhs", q, np.repeat(k, 4, axis=2)) * SCALE
    assert np.allclose(lse, s)


def test_last_row_agrees_with_the_decode_oracle_over_its_rows():
    rng = np.random.default_rng(1)
    n, window, sinks = 40, 7, 3
    q, k, v = _rand(rng, 1, n, 32, 128), _rand(rng, 1, n, 8, 128), _rand(rng, 1, n, 8, 128)
    out, lse = ow.window_attention(q, k, v, [n], window, sinks, SCALE)
    rows = np.r_[0:sinks, n - window:n]
    ref, ref_lse = od.decode_fp64(q[0, -1], k[0, rows], v[0, rows], SCALE)
    assert np.allclose(out[0, -1], ref) and np.allclose(lse[0, :, -1], ref_lse)


def test_padding_rows_are_empty():
    rng = np.random.default_rng(2)
    q, k, v = _rand(rng, 3, 6, 32, 128), _rand(rng, 3, 6, 8, 128), _rand(rng, 3, 6, 8, 128)
    out, lse = ow.window_attention(q, k, v, [0, 2, 6], 3, 1, SCALE)
    assert not out[0].any() and np.isinf(lse[0]).all()
    assert not out[1, 2:].any() and np.isinf(lse[1, :, 2:]).all() and np.isfinite(lse[1, :, :2]).all()


@pytest.mark.parametrize("window,sinks,lens", [(3, 0, None), (2, 2, [5]), (1, 1, None)])
def test_gradients_against_differences(window, sinks, lens):
    rng = np.random.default_rng(3)
    q, k, v = _rand(rng, 1, 7, 32, 128), _rand(rng, 1, 7, 8, 128), _rand(rng, 1, 7, 8, 128)
    g = _rand(rng, 1, 7, 32, 128)
    grads = ow.window_backward(q, k, v, g, lens, window, sinks, SCALE)
    f = lambda: (ow.window_attention(q, k, v, lens, window, sinks, SCALE)[0] * g).sum()  # noqa: E731
    for x, d in zip((q, k, v), grads):
        for _ in range(6):
            at = tuple(rng.integers(0, s) for s in x.shape)
            old, h = x[at], 1e-5
            x[at] = old + h
            up = f()
            x[at] = old - h
            down = f()
            x[at] = old
            assert abs((up - down) / (2 * h) - d[at]) < 1e-7 * max(1, abs(d[at])) + 1e-8
