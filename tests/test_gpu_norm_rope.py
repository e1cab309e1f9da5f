"""Per-head norms with the rotation on the GPU: serving step and training step against the float64 oracle."""
import numpy as np
import pytest
import torch

from oracle import int4 as oi
from oracle import layout as ol
from oracle import norm_rope as on

pytestmark = pytest.mark.gpu
EPS = 1e-6
# fp32 arithmetic: the sum of squares is 128 positive terms in a tree over 8 lanes of 16 (24 roundings), r and the products five
# more, the rotation three: 32 x 2^-24 of the terms' sizes; gradients take two such sums and their products (96)
FWD, BWD = 32 * 2.0 ** -24, 96 * 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _rand(seed, shape, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def _weights(seed, dtype=torch.bfloat16):
    return tuple((1 + 0.3 * _rand(seed + i, (128,), torch.float32)).to(dtype) for i in (0, 1))


def _np(t):
    return t.detach().double().cpu().numpy()


def _fwd_tol(x, w, c, s, eps, half):
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    y = np.abs(x * r * w)
    c, s = np.abs(c), np.abs(s)
    sizes = np.concatenate([y[..., :64] * c + y[..., 64:] * s, y[..., 64:] * c + y[..., :64] * s], -1)
    return (half + FWD) * sizes * 1.01 + 1e-40


def _check_forward(got, x, w, c, s, eps=EPS):
    x, w, c, s = _np(x), _np(w), _np(c), _np(s)
    want = on.forward(x, w, c, s, eps)
    half = HALF[got.dtype]
    err = np.abs(_np(got) - want)
    assert (err <= half * np.abs(want) + _fwd_tol(x, w, c, s, eps, 0.0)).all(), err.max()


def _step(T, seed, int4=False, pool=None):
    from abridgekv_amd import ops
    q, k, v = (_rand(seed + i, (T, h, 128), scale=3.0) for i, h in enumerate((32, 8, 8)))
    pool = pool or -(-T // 16) + 2
    shape = ops.kv_cache_int4_shape(pool) if int4 else ops.kv_cache_shape(pool)
    cache = torch.zeros(shape, dtype=torch.uint8 if int4 else torch.bfloat16, device="cuda")
    slots = torch.from_numpy(np.random.default_rng(seed).permutation(16 * pool)[:T].astype(np.int64))
    slots[2::5] = -1
    return q, k, v, cache, slots


@pytest.mark.parametrize("weights", ["bf16", "f32", None])
@pytest.mark.parametrize("T", [1, 2, 61, 300])
def test_serving_step(T, weights):
    from abridgekv_amd import ops
    q, k, v, cache, slots = _step(T, T)
    wq, wk = (None, None) if weights is None else _weights(T, torch.float32 if weights == "f32" else torch.bfloat16)
    pos = torch.from_numpy(np.random.default_rng(T).integers(0, 5000, T))
    cs = ops.rope_cos_sin_cache(5000)
    dev = [None if t is None else t.cuda() for t in (q, k, v, pos, cs, slots, wq, wk)]
    out = ops.qk_norm_rope_append(*dev[:5], dev[5], cache, q_weight=dev[6], k_weight=dev[7], eps=EPS, max_position=4999)
    assert all(torch.equal(a.cuda(), b) for a, b in zip((q, k, v), dev))              # inputs stay as they are
    c, s = cs[pos][:, None, :64], cs[pos][:, None, 64:]
    rows = cache.view(-1, 2, 16, 8, 128)
    if weights is None:
        q64, k64 = (on.rotate(_np(t), _np(c), _np(s)) for t in (q, k))
        assert (np.abs(_np(out) - q64) <= 2.0 ** -8 * np.abs(q64) + FWD * 30).all()
    else:
        _check_forward(out, q, wq, c, s)
    real = [t for t in range(T) if slots[t] >= 0]
    for t in real:
        row = rows[int(slots[t]) // 16, :, int(slots[t]) % 16]
        assert torch.equal(row[1].cpu(), v[t])
        if weights is not None:
            _check_forward(row[0], k[t], wk, c[t], s[t])
        else:
            assert (np.abs(_np(row[0]) - k64[t]) <= 2.0 ** -8 * np.abs(k64[t]) + FWD * 30).all()
    rows.view(-1)                                            # (the rest of the cache is as it was)
    mask = torch.ones(rows.shape[0], 16, dtype=torch.bool)
    for t in real:
        mask[int(slots[t]) // 16, int(slots[t]) % 16] = False
    assert not rows.transpose(1, 2)[mask.cuda()].any()


def test_serving_step_matches_the_rotation_alone():
    """Without weights: the rows that rope_kv_append writes, bit by bit."""
    from abridgekv_amd import ops
    q, k, v, cache, slots = (t.cuda() for t in _step(40, 3))
    other = cache.clone()
    pos = torch.arange(40, device="cuda") * 3
    cs = ops.rope_cos_sin_cache(600, device="cuda")
    out = ops.qk_norm_rope_append(q, k, v, pos, cs, slots, cache, block_c=64, codes_k=16, max_position=117, code_span=48)
    qr, kr = q.clone(), k.clone()
    ops.rope_kv_append(qr, kr, v, pos, cs, slot_mapping=slots, kv_cache=other, block_c=64, codes_k=16, max_position=117, code_span=48)
    assert torch.equal(out, qr) and torch.equal(cache, other)


def test_serving_step_layout_positions():
    """Bit-reversed code positions of the abridged layout, through the norms."""
    from abridgekv_amd import ops
    q, k, v, cache, slots = _step(200, 4)
    wq, wk = _weights(4)
    logical = torch.arange(37, 237)
    rope = torch.from_numpy(ol.bitrev_rope_positions(logical.numpy(), 64, 16).astype(np.int64))
    cs = ops.rope_cos_sin_cache(200)
    out = ops.qk_norm_rope_append(*(t.cuda() for t in (q, k, v, logical, cs, slots)), cache, q_weight=wq.cuda(), k_weight=wk.cuda(),
                                  block_c=64, codes_k=16, max_position=236)
    _check_forward(out, q, wq, cs[rope][:, None, :64], cs[rope][:, None, 64:])


def test_serving_step_in_place_and_slices():
    """Queries, keys and values as slices of one projection; the outputs over the queries."""
    from abridgekv_amd import ops
    qkv = _rand(6, (50, 48, 128)).cuda()
    wq, wk = (w.cuda() for w in _weights(6))
    _, _, _, cache, slots = _step(50, 6)
    slots, pos, cs = slots.cuda(), torch.arange(50, device="cuda"), ops.rope_cos_sin_cache(50, device="cuda")
    other, before = cache.clone(), qkv.clone()
    want = ops.qk_norm_rope_append(*(qkv[:, a:b].contiguous() for a, b in ((0, 32), (32, 40), (40, 48))), pos, cs, slots, other,
                                   q_weight=wq, k_weight=wk)
    got = ops.qk_norm_rope_append(qkv[:, :32], qkv[:, 32:40], qkv[:, 40:], pos, cs, slots, cache, q_weight=wq, k_weight=wk,
                                  out=qkv[:, :32])
    assert torch.equal(got, want) and torch.equal(cache, other) and torch.equal(qkv[:, 32:], before[:, 32:])


@pytest.mark.parametrize("weights", [True, False])
def test_serving_step_into_4_bits(weights):
    """The rows of the bf16 cache, quantised: byte by byte."""
    from abridgekv_amd import ops
    q, k, v, cache, slots = _step(77, 8)
    _, _, _, small, _ = _step(77, 8, int4=True)
    wq, wk = (w.cuda() for w in _weights(8)) if weights else (None, None)
    q, k, v, slots = (t.cuda() for t in (q, k, v, slots))
    v[5, 2, 40] = float("nan")
    args = (torch.arange(77, device="cuda"), ops.rope_cos_sin_cache(77, device="cuda"), slots)
    a = ops.qk_norm_rope_append(q, k, v, *args, cache, q_weight=wq, k_weight=wk)
    b = ops.qk_norm_rope_append(q, k, v, *args, small, q_weight=wq, k_weight=wk)
    assert torch.equal(a, b)
    host = cache.float().cpu().numpy().transpose(0, 2, 1, 3, 4).reshape(-1, 2, 8, 128)
    got = small.cpu().numpy().transpose(0, 2, 1, 3).reshape(-1, 2, 640)
    for t in slots.tolist():
        if t >= 0:
            assert np.array_equal(got[t], oi.quantise(host[t]))


def test_serving_step_odd_rows():
    """Zero rows stay zero, a NaN reaches its own head row only."""
    from abridgekv_amd import ops
    q, k, v, cache, slots = (t.cuda() for t in _step(4, 9))
    wq, wk = (w.cuda() for w in _weights(9))
    q[1, 3] = 0
    q[2, 7, 5] = float("nan")
    out = ops.qk_norm_rope_append(q, k, v, torch.arange(4, device="cuda"), ops.rope_cos_sin_cache(4, device="cuda"), slots, cache,
                                  q_weight=wq, k_weight=wk)
    assert not out[1, 3].any() and out[2, 7].isnan().all()
    bad = out.isnan().any(-1)
    assert int(bad.sum()) == 1


def _angles(B, S, seed, dtype):
    a = torch.randn((B, S, 64), generator=torch.Generator().manual_seed(seed)) * 3
    a = torch.cat([a, a], -1)
    return a.cos().to(dtype), a.sin().to(dtype)


CASES = [  # B, S, type, angles' batch and type, weights' type
    (1, 1, torch.bfloat16, 1, torch.bfloat16, torch.bfloat16),
    (2, 37, torch.bfloat16, 1, torch.float32, torch.float32),
    (3, 130, torch.bfloat16, 3, torch.bfloat16, torch.bfloat16),
    (1, 5, torch.float32, 1, torch.float32, torch.float32),
    (2, 200, torch.float32, 2, torch.bfloat16, torch.float32),
    (1, 5000, torch.bfloat16, 1, torch.bfloat16, torch.bfloat16),
]


def _check_backward(grad, dw, x, w, c, s, dout):
    x, w64, c, s, g = _np(x), _np(w), _np(c), _np(s), _np(dout)
    dx_want, dw_want = on.backward(x, w64, c, s, EPS, g)
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + EPS)
    ga, gb, ca, sa = np.abs(g[..., :64]), np.abs(g[..., 64:]), np.abs(c), np.abs(s)
    dy = np.concatenate([ga * ca + gb * sa, gb * ca + ga * sa], -1)
    size = r * (dy * np.abs(w64) + np.abs(x) * r * r * (dy * np.abs(w64 * x)).mean(-1, keepdims=True))
    err = np.abs(_np(grad) - dx_want)
    assert (err <= HALF[grad.dtype] * np.abs(dx_want) + BWD * size).all(), (err - HALF[grad.dtype] * np.abs(dx_want)).max()
    # the weights' sums: at most rows / 32 terms in a row in a lane, then trees of 8 rows, 4 waves, 1024 parts (16 apart)
    terms = (dy * np.abs(x) * r).reshape(-1, 128).sum(0)
    n = x.size // 128 / 32 + 100
    assert (np.abs(_np(dw) - dw_want) <= HALF[dw.dtype] * np.abs(dw_want) + n * 2.0 ** -24 * terms).all()


@pytest.mark.parametrize("B,S,dt,ab,adt,wdt", CASES)
def test_training_step(B, S, dt, ab, adt, wdt):
    from abridgekv_amd import fused
    q, k, dq, dk = (_rand(B * S + i, (B, S, h, 128), dt, 2.0) for i, h in enumerate((32, 8, 32, 8)))
    wq, wk = _weights(S, wdt)
    cos, sin = _angles(ab, S, S + 1, adt)
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, wq, wk)]
    qo, ko = fused.qk_norm_rope(leaves[0], leaves[1], cos.cuda(), sin.cuda(), leaves[2], leaves[3], EPS)
    grads = torch.autograd.grad((qo, ko), leaves, (dq.cuda(), dk.cuda()))
    assert qo.dtype == dt and [g.dtype for g in grads] == [dt, dt, wdt, wdt]
    c, s = cos[:, :, None, :64], sin[:, :, None, :64]
    for got, grad, dw, x, w, dout in ((qo, grads[0], grads[2], q, wq, dq), (ko, grads[1], grads[3], k, wk, dk)):
        _check_forward(got, x, w, c, s)
        _check_backward(grad, dw, x, w, c, s, dout)
    again = torch.autograd.grad(fused.qk_norm_rope(leaves[0], leaves[1], cos.cuda(), sin.cuda(), leaves[2], leaves[3], EPS), leaves,
                                (dq.cuda(), dk.cuda()))
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


def test_training_step_views_and_broadcast_gradients():
    """Slices of one projection, gradients that autograd hands over expanded and transposed, a loss of the keys alone."""
    from abridgekv_amd import fused
    qkv = _rand(1, (2, 30, 48, 128)).cuda()
    wq, wk = (w.cuda() for w in _weights(2))
    cos, sin = (t.cuda() for t in _angles(1, 30, 3, torch.bfloat16))
    a = qkv.clone().requires_grad_(True)
    qo, ko = fused.qk_norm_rope(a[:, :, :32], a[:, :, 32:40], cos, sin, wq, wk)
    b = qkv.clone().requires_grad_(True)
    qd, kd = fused.qk_norm_rope(b[:, :, :32].contiguous(), b[:, :, 32:40].contiguous(), cos, sin, wq, wk)
    assert torch.equal(qo, qd) and torch.equal(ko, kd)
    g = _rand(5, (2, 32, 30, 128)).cuda()
    (ga,) = torch.autograd.grad((qo.transpose(1, 2) * g).sum() + ko.sum(), a)
    (gb,) = torch.autograd.grad((qd, kd), b, (g.transpose(1, 2).contiguous(), torch.ones_like(kd)))
    assert torch.equal(ga, gb) and not ga[:, :, 40:].any()
    w = wk.clone().requires_grad_(True)
    _, ko = fused.qk_norm_rope(qkv[:, :, :32], qkv[:, :, 32:40], cos, sin, wq, w)
    ko.float().sum().backward()                              # the queries' gradient is none
    assert w.grad.abs().sum() > 0


def test_training_step_second_derivative_is_refused():
    from abridgekv_amd import fused
    q, k = (_rand(i, (1, 3, h, 128), torch.float32).cuda().requires_grad_(True) for i, h in ((0, 32), (1, 8)))
    wq, wk = (w.cuda() for w in _weights(2, torch.float32))
    cos, sin = (t.cuda() for t in _angles(1, 3, 3, torch.float32))
    qo, _ = fused.qk_norm_rope(q, k, cos, sin, wq, wk)
    (g,) = torch.autograd.grad(qo.square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        g.sum().backward()


def test_empty_batch():
    from abridgekv_amd import fused, ops
    q, k = (torch.empty((2, 0, h, 128), dtype=torch.bfloat16, device="cuda", requires_grad=True) for h in (32, 8))
    wq, wk = (w.cuda().requires_grad_(True) for w in _weights(2))
    cos, sin = (t.cuda() for t in _angles(1, 0, 3, torch.bfloat16))
    qo, ko = fused.qk_norm_rope(q, k, cos, sin, wq, wk)
    grads = torch.autograd.grad((qo, ko), (q, k, wq, wk), (qo.detach(), ko.detach()))
    assert qo.shape == q.shape and not grads[2].any() and not grads[3].any()
    e = torch.empty((0, 32, 128), dtype=torch.bfloat16, device="cuda")
    i = torch.empty(0, dtype=torch.int64, device="cuda")
    cache = torch.zeros(ops.kv_cache_shape(1), dtype=torch.bfloat16, device="cuda")
    assert ops.qk_norm_rope_append(e, e[:, :8], e[:, :8], i, ops.rope_cos_sin_cache(4, device="cuda"), i, cache).shape == e.shape


def test_training_step_captured():
    """Forward and backward of a training step in a graph: replays as the eager calls."""
    from abridgekv_amd import ops
    B, S = 2, 300
    q, k, dq, dk = (_rand(i, (B, S, h, 128)).cuda() for i, h in enumerate((32, 8, 32, 8)))
    wq, wk = (w.cuda() for w in _weights(2))
    cos, sin = (t.cuda() for t in _angles(1, S, 3, torch.bfloat16))

    def step():
        return (*ops.qk_norm_rope(q, k, cos, sin, wq, wk), *ops.qk_norm_rope_backward(q, k, dq, dk, cos, sin, wq, wk))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        q.copy_(_rand(40 + i, q.shape))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step())), i
