"""The 4-bit rows' oracle against the format's words, closed forms and the unquantised decode oracle."""
import numpy as np
import pytest

from oracle import decode as od
from oracle import int4 as oi

RNG = np.random.default_rng(3)


def _rows(n, seed=0):
    return oi.bf16(np.random.default_rng(seed).standard_normal((n, 8, 128)))


def test_places_are_distinct():
    """512 bits of a head's words, each of a dim's four used once; neighbouring dims in the halves of a register."""
    bits = sorted(32 * w + b + i for d in range(128) for w, b in [oi.place(d)] for i in range(4))
    assert bits == list(range(512))
    for d in range(0, 128, 2):
        (w0, b0), (w1, b1) = oi.place(d), oi.place(d + 1)
        assert w0 == w1 and b1 == b0 + 16 and b0 < 16
    for j in range(4):                                       # words 4 j .. + 3: dims 8 j .. + 7 of the four groups
        assert [oi.place(32 * i + 8 * j)[0] for i in range(4)] == [4 * j + i for i in range(4)]


def test_values_are_within_half_a_step():
    """A code is the nearest: half a step, and 15 times the step's own rounding (2^-8 of it) at the
    far end; the minimum is exact."""
    x = _rows(40)
    step, lo, codes = oi.split(oi.quantise(x))
    got = oi.values(oi.quantise(x))
    err = np.abs(got - x).reshape(40, 8, 4, 32)
    assert (err <= step[..., None] * (0.5 + 15 * 2.0 ** -8)).all()
    g = x.reshape(40, 8, 4, 32)
    assert np.array_equal(lo, g.min(-1)) and codes.max() == 15 and codes.min() == 0
    assert (np.abs(np.take_along_axis(got.reshape(g.shape), g.argmin(-1)[..., None], -1)[..., 0] - lo) == 0).all()


def test_closed_forms():
    x = np.zeros((1, 8, 128), np.float32)
    x[0, 0] = 3.0                                            # constant groups
    x[0, 1, :32] = np.arange(32) % 16                        # codes as they are
    x[0, 2, 5] = np.inf
    x[0, 2, 40] = np.nan
    x[0, 3, 0], x[0, 3, 1] = 3e38, -3e38                     # a span that float32 does not hold
    got = oi.values(oi.quantise(x))
    assert (got[0, 0] == 3.0).all() and np.array_equal(got[0, 1], x[0, 1])
    assert np.isnan(got[0, 2, :64]).all() and (got[0, 2, 64:] == 0).all()
    assert np.isnan(got[0, 3, :32]).all() and (got[0, 3, 32:] == 0).all()


def test_bf16_rounding():
    torch = pytest.importorskip("torch")
    x = np.concatenate([RNG.standard_normal(4000).astype(np.float32) * np.float32(s) for s in (1e-39, 1e-3, 1, 5e37)])
    assert np.array_equal(oi.bf16(x), torch.from_numpy(x).to(torch.bfloat16).float().numpy())


def test_attention_is_the_decode_oracles_over_the_values():
    k, v, q = oi.quantise(_rows(50, 1)), oi.quantise(_rows(50, 2)), RNG.standard_normal((1, 32, 128))
    out, lse, tol, ltol = oi.attend(q, k, v, np.ones((1, 50), bool), 0.088)
    want, want_lse = od.decode_fp64(q[0], oi.values(k), oi.values(v), 0.088)
    assert np.allclose(out[0], want, atol=1e-12) and np.allclose(lse[0], want_lse, atol=1e-12)
    assert (tol > 0).all() and (tol < 0.05).all() and (ltol < 1e-2).all()
    vis = np.zeros((2, 50), bool)
    vis[1, :3] = True
    out, lse, _, _ = oi.attend(np.repeat(q, 2, 0), k, v, vis, 0.088)
    assert (out[0] == 0).all() and (lse[0] == -np.inf).all()
    assert np.allclose(out[1], od.decode_fp64(q[0], oi.values(k)[:3], oi.values(v)[:3], 0.088)[0], atol=1e-12)
