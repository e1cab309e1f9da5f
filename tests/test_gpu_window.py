"""Sliding-window attention with sinks on the GPU against the float64 oracle, element by element within the bounds that the
oracle derives from bf16's half step (oracle/window.py)."""
import types

import numpy as np
import pytest
import torch

from oracle import window as ow

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5
BIG = (1 << 31) - 1


def _make(seed, B, S, lens=None, pad=float("nan"), fused=False):
    """q, k, v, dout bf16 on the GPU (padding rows hold ``pad``) and float64 copies with the padding at 0."""
    gen = torch.Generator().manual_seed(seed)
    ts = [torch.randn((B, S, h, 128), generator=gen).to(torch.bfloat16) for h in (32, 8, 8, 32)]
    ref = [t.double().clone() for t in ts]
    if lens is not None:
        for b, n in enumerate(lens):
            for t, r in zip(ts, ref):
                t[b, n:] = pad
                r[b, n:] = 0
    if fused:                                                # q, k, v as views of one [B, S, 48, 128] projection
        qkv = torch.cat(ts[:3], 2).cuda()
        dev = [qkv[:, :, :32], qkv[:, :, 32:40], qkv[:, :, 40:], ts[3].cuda()]
    else:
        dev = [t.cuda() for t in ts]
    return dev, [r.numpy() for r in ref]


def _lens(lens):
    return None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")


# B, S, lens, window, sinks
SHAPES = [
    (1, 1, None, 1, 0), (2, 1, [1, 0], 5, 3), (1, 2, None, 1, 1), (1, 63, None, 7, 2), (1, 64, None, 64, 0),
    (1, 65, None, 64, 1), (2, 130, [130, 65], 1, 0), (1, 200, None, BIG, 0), (1, 200, None, 1, BIG),
    (3, 257, [257, 64, 0], 64, 4), (2, 300, [299, 129], 65, 64), (1, 700, None, 128, 4), (2, 640, None, 63, 130),
    (1, 1000, None, 256, 17), (2, 520, [513, 1], 100, 65),
]


@pytest.mark.parametrize("B,S,lens,window,sinks", SHAPES)
def test_forward(B, S, lens, window, sinks):
    from abridgekv_amd import ops
    (q, k, v, _), ref = _make(S + window % 97, B, S, lens)
    lse = torch.full((B, 32, S), 7.0, device="cuda")
    out, _ = ops.window_attention(q, k, v, window, sinks, seq_lens=_lens(lens), lse=lse)
    want, want_lse, tol = ow.window_attention(*ref[:3], lens, window, sinks, SCALE, bounds=True)
    got = out.double().cpu().numpy()
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= tol).all(), np.abs(got - want).max()
    got_lse = lse.double().cpu().numpy()
    empty = np.isinf(want_lse)
    assert (got_lse[empty] == -np.inf).all()
    # the sum of weights that were rounded by at most half a step each
    assert np.abs(got_lse[~empty] - want_lse[~empty]).max(initial=0) <= ow.SLACK * ow.EPS + 1e-4


@pytest.mark.parametrize("B,S,lens,window,sinks", SHAPES)
def test_forward_fp32(B, S, lens, window, sinks):
    """fp32 mode: 128-term dot products and sums over up to S rows in fp32, |out| <= max|v| of about 4.5: 3e-5 covers a
    score error of 128 x 2^-24 x |q . k| (about 2e-6 relative weight error each) and the sums' rounding."""
    from abridgekv_amd import ops
    (q, k, v, _), ref = _make(S + window % 97, B, S, lens)
    lse = torch.empty((B, 32, S), device="cuda")
    out, _ = ops.window_attention(q.float(), k.float(), v.float(), window, sinks, seq_lens=_lens(lens), lse=lse)
    assert out.dtype == torch.float32
    want, want_lse = ow.window_attention(*ref[:3], lens, window, sinks, SCALE)
    assert np.abs(out.double().cpu().numpy() - want).max() <= 3e-5
    got_lse, empty = lse.double().cpu().numpy(), np.isinf(want_lse)
    assert (got_lse[empty] == -np.inf).all() and np.abs(got_lse[~empty] - want_lse[~empty]).max(initial=0) <= 1e-5


@pytest.mark.parametrize("B,S,lens,window,sinks", SHAPES)
def test_backward(B, S, lens, window, sinks):
    from abridgekv_amd import ops
    (q, k, v, g), ref = _make(S + window % 97, B, S, lens)
    lse = torch.empty((B, 32, S), device="cuda")
    out, _ = ops.window_attention(q, k, v, window, sinks, seq_lens=_lens(lens), lse=lse)
    got = ops.window_attention_backward(q, k, v, out, lse, g, window, sinks, seq_lens=_lens(lens))
    want = ow.window_backward(*ref, lens, window, sinks, SCALE, bounds=True)
    for name, x, d, tol in zip(("dq", "dk", "dv"), got, want[::2], want[1::2]):
        x = x.double().cpu().numpy()
        assert np.isfinite(x).all(), name
        assert (np.abs(x - d) <= tol).all(), (name, np.abs(x - d).max())


def test_far_sink_parts_add_up():
    """Sinks in two key tiles, seen by far query tiles in several parts, against the oracle, twice with the same bits."""
    from abridgekv_amd import ops
    S, window, sinks, lens = 2200, 70, 70, [2200, 1111]
    (q, k, v, g), ref = _make(5, 2, S, lens)
    sl = _lens(lens)
    lse = torch.empty((2, 32, S), device="cuda")
    out, _ = ops.window_attention(q, k, v, window, sinks, seq_lens=sl, lse=lse)
    got = ops.window_attention_backward(q, k, v, out, lse, g, window, sinks, seq_lens=sl)
    again = ops.window_attention_backward(q, k, v, out, lse, g, window, sinks, seq_lens=sl)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    # a slice of heads is enough for the float64 side: KV head 3 and its query heads
    part = [ref[0][:, :, 12:16], ref[1][:, :, 3:4], ref[2][:, :, 3:4], ref[3][:, :, 12:16]]
    want = ow.window_backward(*part, lens, window, sinks, SCALE, bounds=True)
    for name, x, d, tol in zip(("dq", "dk", "dv"), (got[0][:, :, 12:16], got[1][:, :, 3:4], got[2][:, :, 3:4]), want[::2],
                               want[1::2]):
        x = x.double().cpu().numpy()
        assert (np.abs(x - d) <= tol).all(), (name, np.abs(x - d).max())


def test_views_streams_and_given_outputs():
    """Views of one fused projection, [B, heads, S, D] storage, a caller's out and another stream give the same bits."""
    from abridgekv_amd import ops
    (q, k, v, _), _ = _make(3, 2, 150, [150, 77])
    sl = _lens([150, 77])
    base, _ = ops.window_attention(q, k, v, 40, 3, seq_lens=sl)
    (fq, fk, fv, _), _ = _make(3, 2, 150, [150, 77], fused=True)
    assert torch.equal(ops.window_attention(fq, fk, fv, 40, 3, seq_lens=sl)[0], base)
    hq, hk, hv = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v))
    out = torch.empty((2, 32, 150, 128), dtype=torch.bfloat16, device="cuda").transpose(1, 2)
    assert ops.window_attention(hq, hk, hv, 40, 3, seq_lens=sl, out=out)[0] is out and torch.equal(out, base)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other, _ = ops.window_attention(q, k, v, 40, 3, seq_lens=sl)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, base)


def test_autograd_through_the_attention_function():
    from abridgekv_amd.compress_forward import WindowMask, masked_attention_forward
    lens = [90, 200]
    (q, k, v, g), ref = _make(9, 2, 200, lens, pad=0.0)
    qs = [t.transpose(1, 2).requires_grad_(True) for t in (q, k, v)]
    module = types.SimpleNamespace(layer_idx=0)
    out, _ = masked_attention_forward(module, *qs, WindowMask(50, 4, _lens(lens)), scaling=SCALE)
    grads = torch.autograd.grad(out, qs, g)
    want = ow.window_backward(*ref, lens, 50, 4, SCALE, bounds=True)
    for x, d, tol in zip(grads, want[::2], want[1::2]):
        assert (np.abs(x.transpose(1, 2).double().cpu().numpy() - d) <= tol).all()
    # a layer's own sliding window: no sinks, no padding; a broadcast gradient
    out, _ = masked_attention_forward(module, *qs, None, scaling=SCALE, sliding_window=50)
    assert torch.equal(out, masked_attention_forward(module, *qs, WindowMask(50), scaling=SCALE)[0])
    grads = torch.autograd.grad(out.sum(), qs)
    want = ow.window_backward(*(t.detach().transpose(1, 2).double().cpu().numpy() for t in qs), np.ones_like(ref[3]), None,
                              50, 0, SCALE, bounds=True)
    for x, d, tol in zip(grads, want[::2], want[1::2]):
        assert (np.abs(x.transpose(1, 2).double().cpu().numpy() - d) <= tol).all()


def test_graph_replays_match_eager_calls():
    from abridgekv_amd import ops
    (q, k, v, g), _ = _make(13, 2, 900)
    lse = torch.empty((2, 32, 900), device="cuda")

    def call():
        out, _ = ops.window_attention(q, k, v, 80, 20, lse=lse)
        return (out, *ops.window_attention_backward(q, k, v, out, lse, g, 80, 20))

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    for seed in range(4):
        (nq, nk, nv, ng), _ = _make(100 + seed, 2, 900)
        for t, x in zip((q, k, v, g), (nq, nk, nv, ng)):
            t.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        want = call()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), seed


def _paged(rows_k, rows_v, pool, seed, garbage):
    rng = np.random.default_rng(seed)
    need = [-(-r.shape[0] // 16) for r in rows_k]
    pages = rng.permutation(pool)[: sum(need)]
    table = np.zeros((len(need), max(1, max(need))), np.int32)
    cache = torch.full((pool, 2, 16, 8, 128), garbage, dtype=torch.bfloat16)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = pages[at: at + n]
        at += n
        pos = np.arange(rows_k[b].shape[0])
        for i, rows in enumerate((rows_k[b], rows_v[b])):
            cache[torch.from_numpy(table[b, pos // 16].astype(np.int64)), i, torch.from_numpy(pos % 16)] = rows
    return cache.cuda(), torch.from_numpy(table).cuda()


@pytest.mark.parametrize("window,sinks", [(1, 0), (40, 4), (64, 64), (300, 17), (BIG, 0), (5, BIG)])
def test_paged_chunks(window, sinks):
    from abridgekv_amd import ops
    gen = torch.Generator().manual_seed(window % 1000 + sinks % 1000)
    chunk, past = [1, 64, 0, 130, 33], [0, 5, 20, 300, 640]
    k = [torch.randn((c + p, 8, 128), generator=gen).to(torch.bfloat16) for c, p in zip(chunk, past)]
    v = [torch.randn((c + p, 8, 128), generator=gen).to(torch.bfloat16) for c, p in zip(chunk, past)]
    cache, table = _paged(k, v, 120, 1, float("nan"))
    T = sum(chunk)
    q = torch.randn((T + 3, 32, 128), generator=gen).to(torch.bfloat16)
    q_start = np.concatenate([[0], np.cumsum(chunk)])
    out = torch.full((T + 3, 32, 128), 5.0, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((T + 3, 32), 5.0, device="cuda")
    ops.paged_prefill_attention_window(q.cuda(), cache, table, q_start, past, window, sinks, out=out, lse=lse)
    assert (out[T:] == 5).all() and (lse[T:] == 5).all()
    for r, (c, p) in enumerate(zip(chunk, past)):
        if c == 0:
            continue
        a = q_start[r]
        vis = ow.visible(np.arange(p, p + c), p + c, window, sinks)
        want, want_lse, _, tol = ow.attend(q[a: a + c].double().numpy(), k[r].double().numpy(), v[r].double().numpy(), vis,
                                           SCALE, bounds=True)
        assert (np.abs(out[a: a + c].double().cpu().numpy() - want) <= tol).all(), r
        assert np.abs(lse[a: a + c].double().cpu().numpy() - want_lse).max() <= ow.SLACK * ow.EPS + 1e-4, r


def test_more_chunks_than_a_launch_takes():
    """150 requests, some without queries, against each alone."""
    from abridgekv_amd import ops
    gen = torch.Generator().manual_seed(3)
    rng = np.random.default_rng(3)
    chunk, past = rng.integers(0, 4, 150) * rng.integers(1, 30, 150), rng.integers(0, 90, 150)
    k = [torch.randn((c + p, 8, 128), generator=gen).to(torch.bfloat16) for c, p in zip(chunk, past)]
    cache, table = _paged(k, k, 1400, 1, float("nan"))
    q_start = np.concatenate([[0], np.cumsum(chunk)])
    q = torch.randn((int(q_start[-1]), 32, 128), generator=gen).to(torch.bfloat16).cuda()
    lse = torch.empty((q.shape[0], 32), device="cuda")
    out, _ = ops.paged_prefill_attention_window(q, cache, table, q_start, past, 50, 3, lse=lse)
    for r in range(150):
        a, b = int(q_start[r]), int(q_start[r + 1])
        if a < b:
            one = torch.empty((b - a, 32), device="cuda")
            alone, _ = ops.paged_prefill_attention_window(q[a:b], cache, table[r: r + 1], [0, b - a], [past[r]], 50, 3, lse=one)
            assert torch.equal(out[a:b], alone) and torch.equal(lse[a:b], one), r


def test_chunks_in_a_captured_graph():
    """The requests' starts are the capture's, rows and tables are read by each replay."""
    from abridgekv_amd import ops
    gen = torch.Generator().manual_seed(9)
    k = [torch.randn((n, 8, 128), generator=gen).to(torch.bfloat16) for n in (400, 90)]
    cache, table = _paged(k, k, 60, 1, float("nan"))
    q = torch.randn((130, 32, 128), generator=gen).to(torch.bfloat16).cuda()
    args = ([0, 100, 130], [300, 60], 120, 4)
    ops.paged_prefill_attention_window(q, cache, table, *args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = ops.paged_prefill_attention_window(q, cache, table, *args)
    junk = [ops.paged_prefill_attention_window(q, cache, table, [0, 7], [50], 3)[0] for _ in range(3)]
    for i in range(3):
        q.copy_(torch.randn(q.shape, generator=gen).to(torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.paged_prefill_attention_window(q, cache, table, *args)[0]), len(junk)


@pytest.mark.parametrize("B,S,lens,window,sinks", SHAPES)
def test_low_part_of_the_outputs(B, S, lens, window, sinks):
    """out + out_low / 256 is off by what the weights' rounding takes (the forward's bound) and by an eighth (half a step of
    e5m2) of out's own rounding; padding 0; out and lse stay; the gradients keep their bounds."""
    from abridgekv_amd import ops
    (q, k, v, g), ref = _make(S + window % 97, B, S, lens)
    lse, lse0 = (torch.empty((B, 32, S), device="cuda") for _ in range(2))
    low = torch.full((B, S, 32, 128), 7.0, device="cuda").to(torch.float8_e5m2)
    out, _ = ops.window_attention(q, k, v, window, sinks, seq_lens=_lens(lens), lse=lse, out_low=low)
    plain, _ = ops.window_attention(q, k, v, window, sinks, seq_lens=_lens(lens), lse=lse0)
    assert torch.equal(out, plain) and torch.equal(lse, lse0)
    want, _, tol = ow.window_attention(*ref[:3], lens, window, sinks, SCALE, bounds=True)
    left = low.float().double().cpu().numpy() / 256
    err = np.abs(out.double().cpu().numpy() + left - want)
    # (an output whose own rounding is below e5m2's smallest step, 2^-16 / 256, is off by half of that)
    assert (err <= tol - (1 - 1 / 8 - 0.03) * ow.EPS * np.abs(want) + 2.0 ** -25).all(), err.max()
    for b, n in enumerate(lens or []):
        assert not left[b, n:].any()
    got = ops.window_attention_backward(q, k, v, out, lse, g, window, sinks, seq_lens=_lens(lens), out_low=low)
    grads = ow.window_backward(*ref, lens, window, sinks, SCALE, bounds=True)
    for name, x, d, tol in zip(("dq", "dk", "dv"), got, grads[::2], grads[1::2]):
        assert (np.abs(x.double().cpu().numpy() - d) <= tol).all(), name


def test_backward_takes_its_row_sums_from_both_parts():
    """A window of one row: P = 1, so dS = dO . V - dO . (out + out_low / 256) for any out and out_low that are given. dS and dQ
    are rounded (two half steps), the products summed in fp32 (128 terms of each dot product)."""
    from abridgekv_amd import ops
    S, n = 150, 100
    (q, k, v, g), ref = _make(11, 1, S, [n])
    sl = _lens([n])
    lse = torch.empty((1, 32, S), device="cuda")
    ops.window_attention(q, k, v, 1, 0, seq_lens=sl, lse=lse)
    gen = torch.Generator().manual_seed(1)
    out = torch.randn((1, S, 32, 128), generator=gen).to(torch.bfloat16)
    low = (300 * torch.randn((1, S, 32, 128), generator=gen)).to(torch.float8_e5m2)
    out[:, n:], low[:, n:] = float("nan"), float("nan")
    dq, dk, _ = ops.window_attention_backward(q, k, v, out.cuda(), lse, g, 1, 0, seq_lens=sl, out_low=low.cuda())
    rq, rk, rv, rg = (x[0, :n] for x in ref)
    rk, rv = np.repeat(rk, 4, 1), np.repeat(rv, 4, 1)
    total = out.double().numpy()[0, :n] + low.float().double().numpy()[0, :n] / 256
    ds = (rg * (rv - total)).sum(-1, keepdims=True)
    fp32 = 256 * 2.0 ** -24 * (np.abs(rg) * (np.abs(rv) + np.abs(total))).sum(-1, keepdims=True) + ow.FP32 * np.abs(ds)
    err = 2 * ow.SLACK * ow.EPS * np.abs(ds) + fp32
    got = dq.double().cpu().numpy()[0]
    assert (np.abs(got[:n] - SCALE * ds * rk) <= SCALE * err * np.abs(rk)).all() and not got[n:].any()
    want, tol = (SCALE * x.reshape(n, 8, 4, 128).sum(2) for x in (ds * rq, err * np.abs(rq)))
    got = dk.double().cpu().numpy()[0]
    # (dK is rounded as the sum of four heads)
    assert (np.abs(got[:n] - want) <= tol + ow.EPS * np.abs(want)).all() and not got[n:].any()
