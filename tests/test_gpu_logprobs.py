"""Log probabilities of given tokens on the GPU against the float64 oracle."""
import numpy as np
import pytest
import torch

from oracle import logprobs as ol

pytestmark = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _logits(T, V, dt, seed, scale=3.0, banned=0):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn((T, V), generator=gen) * scale).to(dt)
    if banned:
        x[:, torch.randperm(V, generator=gen)[:banned]] = -float("inf")
    t = torch.randint(0, V, (T,), generator=gen)
    return x, t


def _np(t):
    return t.detach().double().cpu().numpy()


def _tol(V, size):
    """fp32: a thread's sums of up to V / 512 terms in a row (one split), a tree over 512 threads and the splits (20), the
    exponentials' arguments and results (their weight is the size of what they are taken of)."""
    return 2.0 ** -24 * (V / 512 + 40 + 16 * size)


def _check(got, x, t, temperature, n):
    X, tn = _np(x), t.cpu().numpy()
    ls, lp, ent = ol.forward(X, tn, temperature)
    V = X.shape[1]
    with np.errstate(all="ignore"):
        p = np.exp(ls)
        spread = np.where(p > 0, p * np.abs(ls), 0).sum(1)
        fin = np.isfinite(lp)
        assert np.array_equal(_np(got.logprob)[~fin], lp[~fin], equal_nan=True)
        assert (np.abs(_np(got.logprob) - lp)[fin] <= _tol(V, spread + np.abs(lp))[fin]).all()
        if got.entropy is not None:
            ok = np.isfinite(ent)
            assert np.array_equal(np.isnan(_np(got.entropy)), ~ok)
            assert (np.abs(_np(got.entropy) - ent)[ok] <= (_tol(V, 4 * spread + 1) * (1 + spread))[ok]).all()
    ids = ol.top(X, n)
    assert got.top_ids.dtype == torch.int64 and np.array_equal(got.top_ids.cpu().numpy(), ids)
    want = np.take_along_axis(ls, ids, 1)
    have = _np(got.top_logprobs)
    fin = np.isfinite(want)
    assert np.array_equal(have[~fin], want[~fin], equal_nan=True)
    size = np.abs(np.where(fin, want, 0)) + np.where(np.isfinite(spread), spread, 0)[:, None]
    assert (np.abs(have[fin] - want[fin]) <= _tol(V, size)[fin]).all()


SIZES = [(1, 1, 1), (3, 2, 2), (1, 7, 3), (5, 8, 8), (2, 31, 20), (4, 257, 32), (1, 4099, 5), (600, 300, 1), (2, 50000, 20),
         (1, 131072, 32), (70, 32003, 0), (515, 5001, 4), (3, 8192, 5)]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,V,n", SIZES)
def test_forward(T, V, n, dt):
    from abridgekv_amd import ops
    x, t = _logits(T, V, dt, T + V, banned=V // 10)
    t[::4] = -100 if V % 2 else V                            # rows without a target
    got = ops.token_logprobs(x.cuda(), t.cuda(), 0.7 if V % 3 else 1.0, top=n)
    _check(got, x, t, 0.7 if V % 3 else 1.0, n)
    again = ops.token_logprobs(x.cuda(), t.cuda(), 0.7 if V % 3 else 1.0, top=n, entropy=False)
    assert again.entropy is None and torch.equal(again.logprob, got.logprob) or got.logprob.isnan().any()
    assert torch.equal(again.top_ids, got.top_ids)


@pytest.mark.parametrize("T,V", [(1, 40000), (2, 9000), (600, 3001)])
@pytest.mark.parametrize("kind", ["equal", "two values", "few finite", "all banned", "runs", "descending"])
def test_ties(kind, T, V):
    """Many equal logits, and rows with fewer finite logits than alternatives: the lowest ids, in order."""
    from abridgekv_amd import ops
    x, t = _logits(T, V, torch.bfloat16, V)
    rng = np.random.default_rng(V)
    if kind == "equal":
        x[:] = 1.5
    elif kind == "two values":
        x[:] = torch.from_numpy(rng.integers(0, 2, (T, V)).astype(np.float32)).to(x.dtype)
    elif kind == "few finite":
        x[:] = -float("inf")
        x[:, [V // 2, 3, V - 1]] = torch.tensor([1.0, 2.0, 1.0], dtype=x.dtype)
        x[0, 5] = -0.0
    elif kind == "all banned":
        x[:] = -float("inf")
    elif kind == "runs":
        x[:] = (torch.arange(V) // 700 % 13).to(x.dtype)
    else:
        x[:] = torch.linspace(40, -40, V).to(x.dtype)
    _check(ops.token_logprobs(x.cuda(), t.cuda(), top=20), x, t, 1.0, 20)


def test_rows_that_are_not_finite():
    """A NaN or +inf makes its own row NaN; alternatives take NaN as the lowest."""
    from abridgekv_amd import ops
    x, t = _logits(5, 9000, torch.float32, 1)
    x[1, 77], x[2, 5] = float("nan"), float("inf")
    x[3] = float("nan")
    got = ops.token_logprobs(x.cuda(), t.cuda(), top=3)
    assert got.logprob.isnan().tolist() == got.entropy.isnan().tolist() == [False, True, True, True, False]
    assert np.array_equal(got.top_ids.cpu().numpy(), ol.top(_np(x), 3))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_masks_of_the_lowest_value(dt):
    """Banned by the type's lowest finite value: as by -inf."""
    from abridgekv_amd import ops
    x, t = _logits(3, 20000, dt, 2, banned=15000)
    low = torch.where(x == -float("inf"), torch.finfo(dt).min, x)
    a, b = (ops.token_logprobs(y.cuda(), t.cuda(), top=4, stats=True) for y in (x, low))
    assert torch.equal(a.entropy, b.entropy) and torch.equal(a.top_ids, b.top_ids) and torch.equal(a.stats, b.stats)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_strided_rows(dt):
    """Rows of a wider tensor at every alignment, and results that do not depend on it."""
    from abridgekv_amd import ops
    for off in range(9):
        wide, t = _logits(7, 1234, dt, off)
        wide, t = wide.cuda(), t.cuda() % 1200
        x = wide[:, off: off + 1201]
        got = ops.token_logprobs(x, t, top=5, stats=True)
        _check(got, x, t, 1.0, 5)
        g = torch.ones(7, device="cuda")
        grad = torch.full((7, 1300), 9.0, dtype=dt, device="cuda")
        ops.token_logprobs_backward(x, t, got.stats, g, g, out=grad[:, 3: 1204])
        want = ops.token_logprobs_backward(x.contiguous(), t, got.stats, g, g)
        assert torch.equal(grad[:, 3: 1204], want) and (grad[:, :3] == 9).all() and (grad[:, 1204:] == 9).all()


def _check_grad(grad, x, t, g, h, temperature):
    X, tn = _np(x), t.cpu().numpy()
    want = ol.backward(X, tn, _np(g), _np(h), temperature)
    ls, _, ent = ol.forward(X, tn, temperature)
    p = np.exp(ls)
    lsf = np.where(p > 0, np.abs(ls), 0)
    spread = (p * lsf).sum(1, keepdims=True)
    real = (tn >= 0) & (tn < X.shape[1])
    size = (np.where(real, np.abs(_np(g)), 0)[:, None] + np.abs(_np(h))[:, None] * (lsf + ent[:, None])) / temperature
    hit = np.zeros_like(p)
    hit[np.arange(len(p))[real], tn[real]] = np.abs(_np(g))[real] / temperature
    tol = HALF[grad.dtype] * np.abs(want) + _tol(X.shape[1], lsf + 4 * spread + 2) * p * size * 4 + 2.0 ** -22 * hit + 1e-38
    err = np.abs(_np(grad) - want)
    assert (err <= tol).all(), (err - tol).max()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,V", [(1, 1), (3, 9), (5, 1000), (2, 40001), (130, 3007)])
def test_gradient(T, V, dt):
    from abridgekv_amd import fused
    x, t = _logits(T, V, dt, T * V, banned=V // 10)
    t[::3] = -100
    g, h = (torch.randn(T, generator=torch.Generator().manual_seed(i)) for i in (1, 2))
    leaf = x.cuda().requires_grad_(True)
    lp, ent = fused.token_logprobs(leaf, t.cuda(), 0.8)
    (grad,) = torch.autograd.grad((lp, ent), leaf, (g.cuda(), h.cuda()))
    assert grad.dtype == dt
    _check_grad(grad, x, t, g, h, 0.8)
    zero = torch.zeros(T)
    (only,) = torch.autograd.grad(fused.token_logprobs(leaf, t.cuda(), 0.8)[0].sum(), leaf)
    _check_grad(only, x, t, torch.ones(T), zero, 0.8)
    (only,) = torch.autograd.grad(fused.token_logprobs(leaf, t.cuda(), 0.8)[1].sum(), leaf)
    _check_grad(only, x, t, zero, torch.ones(T), 0.8)


def test_gradient_of_a_banned_target():
    """A target of probability 0: log probability -inf, a finite gradient."""
    from abridgekv_amd import ops
    x, t = _logits(2, 500, torch.float32, 3)
    x[0, t[0]] = -float("inf")
    got = ops.token_logprobs(x.cuda(), t.cuda(), stats=True)
    assert got.logprob[0] == -float("inf")
    g = torch.ones(2)
    _check_grad(ops.token_logprobs_backward(x.cuda(), t.cuda(), got.stats, g.cuda(), None), x, t, g, torch.zeros(2), 1.0)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_gradient_at_a_low_temperature(dt):
    """Banned tokens take exactly no gradient, however steep the others' are."""
    from abridgekv_amd import ops
    x, t = _logits(3, 700, dt, 5, banned=60)
    x[1, 3] = torch.finfo(dt).min
    st = ops.token_logprobs(x.cuda(), t.cuda(), 1e-6, stats=True).stats
    h = torch.full((3,), 1000.0, device="cuda")
    grad = ops.token_logprobs_backward(x.cuda(), t.cuda(), st, h, h, 1e-6).cpu()
    banned = x < -1e25
    banned[torch.arange(3), t] = False
    assert torch.isfinite(grad).all() and banned.any() and not grad[banned].any()


def test_gradient_over_the_logits():
    from abridgekv_amd import ops
    x, t = _logits(9, 4001, torch.bfloat16, 3)
    x, t = x.cuda(), t.cuda()
    st = ops.token_logprobs(x, t, stats=True).stats
    g = torch.randn(9, device="cuda")
    want = ops.token_logprobs_backward(x, t, st, g, g)
    assert torch.equal(ops.token_logprobs_backward(x, t, st, g, g, out=x), want) and torch.equal(x, want)


def test_second_derivative_is_refused():
    from abridgekv_amd import fused
    x, t = _logits(2, 50, torch.float32, 3)
    leaf = x.cuda().requires_grad_(True)
    (g,) = torch.autograd.grad(fused.token_logprobs(leaf, t.cuda())[0].sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        g.square().sum().backward()


def test_offsets_past_32_bits():
    """Rows beyond 4 GiB of logits, forward and backward."""
    from abridgekv_amd import ops
    V, T = 131072, 17000
    x = torch.zeros((T, V), dtype=torch.bfloat16, device="cuda")
    row, t1 = _logits(1, V, torch.bfloat16, 5)
    x[-1] = row[0].cuda()
    t = torch.full((T,), -100, device="cuda")
    t[-1] = int(t1)
    got = ops.token_logprobs(x, t, top=2, stats=True)
    _check(got._replace(**{f: getattr(got, f)[-1:] for f in got._fields}), row, t1, 1.0, 2)
    assert torch.allclose(got.entropy[:-1], torch.full((T - 1,), float(np.log(V)), device="cuda"), rtol=1e-5)
    g = torch.ones(T, device="cuda")
    ops.token_logprobs_backward(x, t, got.stats, g, None, out=x)
    _check_grad(x[-1:], row, t1, torch.ones(1), torch.zeros(1), 1.0)
    assert not x[0].any()


def test_captured():
    from abridgekv_amd import ops
    x, t = _logits(3, 20000, torch.bfloat16, 3)
    x, t = x.cuda(), t.cuda()
    g = torch.ones(3, device="cuda")

    def step():
        got = ops.token_logprobs(x, t, 0.9, top=5, stats=True)
        return (*got, ops.token_logprobs_backward(x, t, got.stats, g, g, 0.9))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        new, nt = _logits(3, 20000, torch.bfloat16, 30 + i)
        x.copy_(new)
        t.copy_(nt)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step())), i
