"""Decode under a window, accumulated weights and eviction on the GPU against the float64 oracles, and a run of them."""
import numpy as np
import pytest
import torch

from oracle import evict as oe
from oracle import window as ow

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5
BIG = (1 << 31) - 1
# A weight exp(s - lse) in fp32: s of 128 products summed in fp32 (|s| <= ~16, 128 x 2^-24 relative to sum |q k| x scale,
# about 1e-5), one exp2 and one division; summed over 4 heads (and queries)
W_TOL = 4e-5


def _paged(lens, seed, garbage=float("nan"), extra_pages=5):
    """Rows k, v [n, 8, 128] of each sequence in a cache of scattered pages whose other rows hold ``garbage``."""
    rng = np.random.default_rng(seed)
    gen = torch.Generator().manual_seed(seed)
    k = [torch.randn((n, 8, 128), generator=gen).to(torch.bfloat16) for n in lens]
    v = [torch.randn((n, 8, 128), generator=gen).to(torch.bfloat16) for n in lens]
    need = [-(-n // 16) for n in lens]
    pool = sum(need) + extra_pages
    pages = rng.permutation(pool)[: sum(need)]
    table = np.zeros((len(lens), max(1, max(need))), np.int32)
    cache = torch.full((pool, 2, 16, 8, 128), garbage, dtype=torch.bfloat16)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = pages[at: at + n]
        at += n
        pos = np.arange(lens[b])
        for i, rows in enumerate((k[b], v[b])):
            cache[torch.from_numpy(table[b, pos // 16].astype(np.int64)), i, torch.from_numpy(pos % 16)] = rows
    q = torch.randn((len(lens), 32, 128), generator=gen).to(torch.bfloat16)
    return q, k, v, cache.cuda(), torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32).cuda()


def _close(out, lse, q, k, v, vis):
    """Decode outputs of one sequence. Split partials are fp16 (2^-11 relative to the split's largest |out|, itself at most
    max|v| of its rows) beside the bounds of the bf16 weights and output."""
    want, want_lse, _, tol = ow.attend(q.double().numpy()[None], k.double().numpy(), v.double().numpy(), vis[None], SCALE, True)
    tol = tol + 2.0 ** -11 * np.abs(v.double().numpy()).max(initial=0)
    assert (np.abs(out.double().cpu().numpy() - want[0]) <= tol[0]).all(), np.abs(out.double().cpu().numpy() - want[0]).max()
    if vis.any():
        assert np.abs(lse.double().cpu().numpy() - want_lse[0]).max() <= 1e-4
    else:
        assert not out.any() and (lse == -np.inf).all()


LENS = [0, 1, 15, 16, 17, 33, 100, 511, 513, 1300]


@pytest.mark.parametrize("split_pages", [2, 8, 32])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 16), (17, 4), (64, 0), (100, 33), (512, 5), (BIG, 0), (3, BIG)])
def test_decode_window(window, sinks, split_pages):
    from abridgekv_amd import ops
    q, k, v, cache, table, sl = _paged(LENS, window % 1000 + sinks % 1000)
    lse = torch.empty((len(LENS), 32), device="cuda")
    out, _ = ops.decode_attention_window(q.cuda(), cache, table, sl, window, sinks, lse=lse, split_pages=split_pages)
    for b, n in enumerate(LENS):
        _close(out[b], lse[b], q[b], k[b], v[b], ow.visible([n - 1], n, window, sinks)[0] if n else np.zeros(0, bool))


def test_decode_window_reads_only_its_pages():
    """Pages between the sinks and the window hold NaN, and their table entries point out of the cache: the same bits."""
    from abridgekv_amd import ops
    q, k, v, cache, table, sl = _paged([1000, 777], 3)
    want, _ = ops.decode_attention_window(q.cuda(), cache, table, sl, 90, 20)
    t = table.clone()
    t[0, 2: (1000 - 90) // 16] = 1 << 30
    t[1, 2: (777 - 90) // 16] = -5
    got, _ = ops.decode_attention_window(q.cuda(), cache, t, sl, 90, 20)
    assert torch.equal(want, got)


def test_decode_window_of_a_prompts_last_row():
    """The last row of the prompt form, within one more rounding of the output."""
    from abridgekv_amd import ops
    q, k, v, cache, table, sl = _paged([700], 11)
    out, _ = ops.decode_attention_window(q.cuda(), cache, table, sl, 128, 4)
    qs = torch.zeros((1, 700, 32, 128), dtype=torch.bfloat16)
    qs[0, -1] = q[0]
    full, _ = ops.window_attention(qs.cuda(), k[0][None].cuda(), v[0][None].cuda(), 128, 4)
    vis = ow.visible([699], 700, 128, 4)
    tol = ow.attend(q.double().numpy(), k[0].double().numpy(), v[0].double().numpy(), vis, SCALE, True)[3][0]
    assert (np.abs((out[0] - full[0, -1]).double().cpu().numpy()) <= 2 * tol + 2.0 ** -11 * 5).all()


def test_decode_more_sequences_than_share_splits():
    """The kernel forms of larger batches (one wave per split)."""
    from abridgekv_amd import ops
    lens = [int(x) for x in np.random.default_rng(5).integers(1, 900, 40)]
    q, k, v, cache, table, sl = _paged(lens, 21)
    M = table.shape[1] * 16
    lse = torch.empty((len(lens), 32), device="cuda")
    out, _ = ops.decode_attention_window(q.cuda(), cache, table, sl, 200, 9, lse=lse, split_pages=4)
    for b in (0, 7, 19, 39):
        _close(out[b], lse[b], q[b], k[b], v[b], ow.visible([lens[b] - 1], lens[b], 200, 9)[0])
    scores = torch.zeros((len(lens), 8, M), device="cuda")
    out, _ = ops.decode_attention_scored(q.cuda(), cache, table, sl, scores, lse=lse, split_pages=4)
    for b in (0, 7, 19, 39):
        _close(out[b], lse[b], q[b], k[b], v[b], np.ones(lens[b], bool))
        w = oe.weights(q[b: b + 1].double().numpy(), k[b].double().numpy(), v[b].double().numpy(), [lens[b] - 1], SCALE)
        assert np.abs(scores[b, :, : lens[b]].double().cpu().numpy() - w).max() <= W_TOL


@pytest.mark.parametrize("B,most", [(24, 4096), (30, 700), (16, 512), (17, 513), (5, 320), (5, 321), (1, 1), (26, 4097)])
def test_decode_scored_whole_and_split(B, most):
    """Sizes on both sides of the rule that picks a workgroup per sequence and head or splits."""
    from abridgekv_amd import ops
    rng = np.random.default_rng(B + most)
    lens = [most] + [int(x) for x in rng.integers(0, min(most, 600), B - 1)] if B > 1 else [most]
    q, k, v, cache, table, sl = _paged(lens, B)
    M = table.shape[1] * 16
    scores = torch.full((B, 8, M), 0.5, device="cuda")
    lse = torch.empty((B, 32), device="cuda")
    out, _ = ops.decode_attention_scored(q.cuda(), cache, table, sl, scores, lse=lse)
    for b in {0, 1 % B, B // 2, B - 1}:
        n = lens[b]
        _close(out[b], lse[b], q[b], k[b], v[b], np.ones(n, bool))
        assert (scores[b, :, n:] == 0.5).all()
        if n:
            w = oe.weights(q[b: b + 1].double().numpy(), k[b].double().numpy(), v[b].double().numpy(), [n - 1], SCALE)
            assert np.abs(scores[b, :, :n].double().cpu().numpy() - 0.5 - w).max() <= W_TOL


@pytest.mark.parametrize("split_pages", [2, 32])
def test_decode_scored(split_pages):
    from abridgekv_amd import ops
    q, k, v, cache, table, sl = _paged(LENS, 7)
    M = table.shape[1] * 16
    start = torch.rand((8, len(LENS), M + 5), generator=torch.Generator().manual_seed(1)).cuda()
    scores = start.clone().permute(1, 0, 2)                  # sequences inside heads, rows longer than needed
    lse = torch.empty((len(LENS), 32), device="cuda")
    out, _ = ops.decode_attention_scored(q.cuda(), cache, table, sl, scores, lse=lse, split_pages=split_pages)
    plain, _ = ops.decode_attention(q.cuda(), cache, table, sl, SCALE, split_pages=split_pages)
    for b, n in enumerate(LENS):
        _close(out[b], lse[b], q[b], k[b], v[b], np.ones(n, bool))
        got = (scores[b] - start.permute(1, 0, 2)[b]).double().cpu().numpy()
        assert not got[:, n:].any()
        if n:
            w = oe.weights(q[b: b + 1].double().numpy(), k[b].double().numpy(), v[b].double().numpy(), [n - 1], SCALE)
            assert np.abs(got[:, :n] - w).max() <= W_TOL + 4 * 2.0 ** -24
    again = start.clone().permute(1, 0, 2)
    ops.decode_attention_scored(q.cuda(), cache, table, sl, again, split_pages=split_pages)
    assert torch.equal(again, scores)
    assert (out - plain).abs().max() <= 2.0 ** -7 * 5        # the same sums but for the partials' rounding


@pytest.mark.parametrize("chunk,past", [([1], [0]), ([64], [0]), ([65, 3], [0, 200]), ([130, 0, 17, 300], [5, 9, 64, 31])])
def test_prefill_scores(chunk, past):
    from abridgekv_amd import ops
    lens = [c + p for c, p in zip(chunk, past)]
    _, k, v, cache, table, _ = _paged(lens, sum(lens))
    gen = torch.Generator().manual_seed(4)
    T = sum(chunk)
    q = torch.randn((T + 2, 32, 128), generator=gen).to(torch.bfloat16)
    q_start = np.concatenate([[0], np.cumsum(chunk)])
    lse = torch.full((T + 2, 32), -float("inf"))
    want = []
    for r, (c, p) in enumerate(zip(chunk, past)):
        a = q_start[r]
        if c == 0:
            want.append(0.0)
            continue
        args = [q[a: a + c].double().numpy(), k[r].double().numpy(), v[r].double().numpy()]
        vis = ow.visible(np.arange(p, p + c), p + c, BIG, 0)
        lse[a: a + c] = torch.from_numpy(ow.attend(*args, vis, SCALE)[1]).float()
        want.append(oe.weights(*args, np.arange(p, p + c), SCALE))
    start = torch.rand((len(chunk), 8, table.shape[1] * 16), generator=gen).cuda()
    scores = start.clone()
    ops.paged_prefill_scores(q.cuda(), cache, table, q_start, past, lse.cuda(), scores)
    for r, n in enumerate(lens):
        got = (scores[r] - start[r]).double().cpu().numpy()
        n = n if chunk[r] else 0
        assert not got[:, n:].any()
        if n:
            # a score of up to 4 x queries is stored in fp32 (and was added to one)
            assert (np.abs(got[:, :n] - want[r]) <= W_TOL * (1 + want[r])).all(), np.abs(got[:, :n] - want[r]).max()


@pytest.mark.parametrize("held", [1.0, float("inf"), float("nan")])
def test_prefill_scores_of_rows_that_see_nothing(held):
    """Rows with lse -inf, whatever they hold, among others and at a request's end, add nothing."""
    from abridgekv_amd import ops
    q, k, v, cache, table, _ = _paged([300], 8)
    q = torch.randn((200, 32, 128), generator=torch.Generator().manual_seed(5)).to(torch.bfloat16).cuda()
    lse = torch.full((200, 32), 6.0, device="cuda")
    want = torch.zeros((1, 8, table.shape[1] * 16), device="cuda")
    got = want.clone()
    dead = torch.zeros(200, dtype=torch.bool)
    dead[[0, 3, 17, 64, 65, 130, 199]] = True
    for at in range(200):                                    # each live row alone, behind its own rows
        if not dead[at]:
            ops.paged_prefill_scores(q[at: at + 1], cache, table, [0, 1], [100 + at], lse[at: at + 1].contiguous(), want)
    q[dead], lse[dead] = held, -float("inf")
    ops.paged_prefill_scores(q, cache, table, [0, 200], [100], lse, got)
    # the same terms added up in other orders: at most 4 x 193 of them
    assert (got - want).abs().max() <= 772 * 2.0 ** -24 * want.max()


def test_prefill_scores_of_more_than_a_launch_takes():
    """150 requests, and 12 of more tiles than one launch lists (over the same pages), against each alone."""
    from abridgekv_amd import ops
    rng = np.random.default_rng(3)
    short = (rng.integers(0, 4, 150) * rng.integers(1, 30, 150), rng.integers(0, 90, 150), 1)
    for chunk, past, seed in (short, (rng.integers(1, 100, 12), rng.integers(8000, 8100, 12), 2)):
        lens = [int(c + p) for c, p in zip(chunk, past)]
        _, k, v, cache, table, _ = _paged(lens if seed == 1 else [8200], seed)
        table = table.expand(len(lens), -1).contiguous()
        q_start = np.concatenate([[0], np.cumsum(chunk)])
        T = int(q_start[-1])
        q = torch.randn((T, 32, 128), generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda()
        lse = torch.full((T, 32), 6.0, device="cuda")
        scores = torch.rand((len(lens), 8, table.shape[1] * 16), device="cuda")
        want = scores.clone()
        ops.paged_prefill_scores(q, cache, table, q_start, past, lse, scores)
        for r in range(len(lens)):
            a, b = int(q_start[r]), int(q_start[r + 1])
            ops.paged_prefill_scores(q[a:b], cache, table[r: r + 1], [0, b - a], [past[r]], lse[a:b], want[r: r + 1])
        # tiles of 64 or 128 keys by the call's sizes: two orders of the same sums
        assert ((scores - want).abs() <= 4 * chunk.max() * 2.0 ** -24 * want).all()


def test_prefill_scores_in_a_captured_graph():
    """The requests' starts are the capture's; queries, lse and scores are each replay's."""
    from abridgekv_amd import ops
    _, k, v, cache, table, _ = _paged([400, 90], 8)
    gen = torch.Generator().manual_seed(2)
    q = torch.randn((130, 32, 128), generator=gen).to(torch.bfloat16).cuda()
    lse = torch.full((130, 32), 6.0, device="cuda")
    scores = torch.zeros((2, 8, 400), device="cuda")
    want = torch.zeros_like(scores)
    ops.paged_prefill_scores(q, cache, table, [0, 100, 130], [300, 60], lse, scores.clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_prefill_scores(q, cache, table, [0, 100, 130], [300, 60], lse, scores)
    for i in range(3):
        q.copy_(torch.randn(q.shape, generator=gen).to(torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        ops.paged_prefill_scores(q, cache, table, [0, 100, 130], [300, 60], lse, want)
        assert torch.equal(scores, want)


def _evict_case(lens, seed, layers=2, levels=None, recorded=False):
    """Caches of rows that name themselves, scores (``levels``: few different ones) and positions."""
    q, k, v, cache, table, sl = _paged(lens, seed, garbage=3.0)
    rng = np.random.default_rng(seed)
    M = table.shape[1] * 16
    shape = (layers, len(lens), 8, M)
    scores = rng.integers(0, levels, shape).astype(np.float32) if levels else rng.lognormal(0, 2, shape).astype(np.float32)
    positions = np.full(shape, -1, np.int32)
    tokens = np.array(lens, np.int32)
    if recorded:                                             # rows of earlier evictions, out of order, 40 tokens gone
        tokens += 40
        for idx in np.ndindex(shape[:3]):
            n = lens[idx[1]]
            old = n * 2 // 3
            positions[idx][:old] = rng.permutation(tokens[idx[1]] - (n - old))[:old] if old else []
    caches = [cache.clone().normal_() for _ in range(layers)]
    return caches, table, sl, scores, positions, tokens


def _check_evict(caches, table, sl, scores, positions, tokens, budget, sinks, recent, **kw):
    from abridgekv_amd import ops
    before = [c.cpu() for c in caches]
    s, p = torch.from_numpy(scores).cuda(), torch.from_numpy(positions).cuda()
    lens = ops.kv_evict(caches, table, sl, s, p, torch.from_numpy(tokens).cuda(), budget, sinks, recent, **kw)
    tab = table.cpu().numpy()
    for layer, cache in enumerate(caches):
        want = before[layer].clone()
        for b, n in enumerate(sl.tolist()):
            assert int(lens[b]) == min(n, budget)
            for h in range(8):
                got = oe.evict(scores[layer, b, h, :n], positions[layer, b, h, :n], int(tokens[b]), budget, sinks, recent)
                moves, ws, wp = got or ([], scores[layer, b, h, :n], positions[layer, b, h, :n])
                for src, dst in moves:
                    want[tab[b, dst // 16], :, dst % 16, h] = before[layer][tab[b, src // 16], :, src % 16, h]
                assert np.array_equal(s[layer, b, h, :n].cpu().numpy(), ws, equal_nan=True), (layer, b, h)
                assert (p[layer, b, h, :n].cpu().numpy() == wp).all(), (layer, b, h)
                assert np.array_equal(s[layer, b, h, n:].cpu().numpy(), scores[layer, b, h, n:], equal_nan=True)
                assert (p[layer, b, h, n:].cpu().numpy() == positions[layer, b, h, n:]).all()
        assert torch.equal(cache.cpu(), want), layer
    return lens


@pytest.mark.parametrize("budget,sinks,recent", [(1, 0, 0), (1, 1, 0), (16, 4, 8), (64, 0, 64), (100, 7, 30), (299, 4, 200),
                                                 (300, 0, 0), (5000, 4, 100)])
@pytest.mark.parametrize("levels,recorded", [(None, False), (3, False), (1, True), (None, True)])
def test_evict(budget, sinks, recent, levels, recorded):
    lens = [0, 1, 15, 16, 63, 64, 65, 300]
    _check_evict(*_evict_case(lens, budget + (levels or 0), levels=levels, recorded=recorded), budget, sinks, recent)


@pytest.mark.parametrize("most,budget", [(300, 100), (1024, 700), (1040, 999)])
def test_evict_many_sequences(most, budget):
    """Enough workgroups for the forms of fewer waves."""
    lens = [most] + [int(x) for x in np.random.default_rng(most).integers(0, min(most, 320), 64)]
    _check_evict(*_evict_case(lens, most, layers=2, levels=200), budget, 3, 40)


def test_evict_odd_scores():
    """NaN, infinities, both zeros and negative scores; ties of all kinds."""
    case = list(_evict_case([200, 130], 9, layers=1))
    odd = np.array([np.nan, np.inf, -np.inf, 0.0, -0.0, 1.0, -1.0, 1e-45, 3e38], np.float32)
    case[3] = odd[np.random.default_rng(2).integers(0, len(odd), case[3].shape)]
    _check_evict(*case, 70, 3, 9)


@pytest.mark.parametrize("n,budget", [(4096, 2048), (4100, 4099), (9000, 2048), (9001, 8000)])
def test_evict_longer_sequences(n, budget):
    _check_evict(*_evict_case([n, 50], n, layers=1, levels=50), budget, 4, 256)


def test_evict_rows_past_lds():
    """A table wider than LDS holds keys for: the keys and lists lie in the workspace."""
    caches, table, sl, scores, positions, tokens = _evict_case([700, 300], 4, layers=1, recorded=True)
    W = 2049
    wide = torch.zeros((2, W), dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table
    pad = ((0, 0), (0, 0), (0, 0), (0, W * 16 - scores.shape[3]))
    _check_evict(caches, wide, sl, np.pad(scores, pad, constant_values=2.0), np.pad(positions, pad, constant_values=7), tokens,
                 256, 4, 60)


def test_evict_by_max_pages_on_a_stream_in_a_graph():
    """max_pages below the table's width, another stream, and replays of a captured call against eager ones."""
    from abridgekv_amd import ops
    caches, table, sl, scores, positions, tokens = _evict_case([400, 350, 90], 6)
    wide = torch.zeros((3, 40), dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table
    pad = ((0, 0), (0, 0), (0, 0), (0, 640 - scores.shape[3]))
    scores, positions = np.pad(scores, pad), np.pad(positions, pad, constant_values=-1)
    _check_evict([c.clone() for c in caches], wide, sl, scores.copy(), positions.copy(), tokens, 200, 2, 50,
                 max_pages=table.shape[1])
    s, p, t = torch.from_numpy(scores).cuda(), torch.from_numpy(positions).cuda(), torch.from_numpy(tokens).cuda()
    keep = [c.clone() for c in caches]
    held = [c.clone() for c in caches]
    hs, hp = s.clone(), p.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.kv_evict(held, wide, sl, hs.clone(), hp.clone(), t, 200, 2, 50)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lens = ops.kv_evict(held, wide, sl, hs, hp, t, 200, 2, 50)
    for i in range(3):
        new = torch.rand(s.shape, generator=torch.Generator().manual_seed(i)).cuda()
        for a, b in zip(held, keep):
            a.copy_(b)
        hs.copy_(new)
        hp.copy_(p)
        lens.zero_()
        graph.replay()
        torch.cuda.synchronize()
        mine, ms, mp = [c.clone() for c in keep], new.clone(), p.clone()
        want = ops.kv_evict(mine, wide, sl, ms, mp, t, 200, 2, 50)
        assert torch.equal(lens, want) and torch.equal(hs, ms) and torch.equal(hp, mp)
        assert all(torch.equal(a, b) for a, b in zip(held, mine))


def test_graph_replays_of_a_scored_step():
    from abridgekv_amd import ops
    lens = [500, 33, 1200]
    q, k, v, cache, table, sl = _paged(lens, 13)
    qd = q.cuda()
    scores = torch.zeros((3, 8, table.shape[1] * 16), device="cuda")
    lse = torch.empty((3, 32), device="cuda")
    ops.decode_attention_scored(qd, cache, table, sl, scores.clone(), lse=lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = ops.decode_attention_scored(qd, cache, table, sl, scores, lse=lse)
        wout, _ = ops.decode_attention_window(qd, cache, table, sl, 300, 7)
    want = torch.zeros_like(scores)
    for i in range(3):
        qd.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        eager, _ = ops.decode_attention_scored(qd, cache, table, sl, want)
        assert torch.equal(out, eager) and torch.equal(scores, want)
        assert torch.equal(wout, ops.decode_attention_window(qd, cache, table, sl, 300, 7)[0])


def test_a_bounded_cache_in_use():
    """Prompt, eviction, decode steps with scores, eviction again: two layers' caches and states against the same run kept in
    float64 lists. The rows each side keeps are compared where the scores' gap exceeds what fp32 can move."""
    from abridgekv_amd import ops
    rng = np.random.default_rng(0)
    gen = torch.Generator().manual_seed(0)
    B, budget, sinks, recent, grow, rounds = 2, 96, 4, 24, 20, 3
    prompt = [130, 90]
    W = -(-(max(max(prompt), budget + grow) + 1) // 16)
    table = torch.from_numpy(rng.permutation(B * W).reshape(B, W).astype(np.int32)).cuda()
    cache = torch.zeros((B * W, 2, 16, 8, 128), dtype=torch.bfloat16, device="cuda")
    M = W * 16
    scores = torch.zeros((1, B, 8, M), device="cuda")
    positions = torch.full((1, B, 8, M), -1, dtype=torch.int32, device="cuda")
    total = np.array(prompt)
    fed = max(prompt) + grow * rounds
    k = torch.randn((B, fed, 8, 128), generator=gen).to(torch.bfloat16)
    v = torch.randn((B, fed, 8, 128), generator=gen).to(torch.bfloat16)

    def append(rows):                                        # rows [(b, slot, token)]
        slots = torch.tensor([int(table[b, s // 16]) * 16 + s % 16 for b, s, _ in rows], dtype=torch.int64, device="cuda")
        ops.kv_append(torch.stack([k[b, t] for b, _, t in rows]).cuda(), torch.stack([v[b, t] for b, _, t in rows]).cuda(),
                      slots, cache)

    append([(b, i, i) for b in range(B) for i in range(prompt[b])])
    T = sum(prompt)
    q = torch.randn((T, 32, 128), generator=gen).to(torch.bfloat16)
    q_start = np.concatenate([[0], np.cumsum(prompt)])
    lse = torch.empty((T, 32), device="cuda")
    ops.paged_prefill_attention(q.cuda(), cache, table, q_start, [0] * B, prompt, True, lse=lse)
    ops.paged_prefill_scores(q.cuda(), cache, table, q_start, [0] * B, lse, scores[0])
    # the same state in float64: per (b, h) a list of [token, weight] in slot order
    state = {}
    for b in range(B):
        w = oe.weights(q[q_start[b]: q_start[b + 1]].double().numpy(), k[b, : prompt[b]].double().numpy(),
                       v[b, : prompt[b]].double().numpy(), np.arange(prompt[b]), SCALE)
        for h in range(8):
            state[b, h] = [[t, w[h, t]] for t in range(prompt[b])]
    lens = torch.tensor(prompt, dtype=torch.int32, device="cuda")
    for _ in range(rounds):
        lens = ops.kv_evict([cache], table, lens, scores, positions, torch.tensor(total, dtype=torch.int32, device="cuda"),
                            budget, sinks, recent)
        for (b, h), rows in state.items():
            n = len(rows)
            got = oe.evict([r[1] for r in rows], [r[0] for r in rows], int(total[b]), budget, sinks, recent)
            if got is not None:
                # tokens that the GPU kept: the same up to scores closer than the weights' errors
                mine = set(positions[0, b, h, :budget].tolist())
                theirs = set(int(x) for x in got[2][:budget])
                edge = {t: x for t, x in rows}
                if mine != theirs:
                    assert len(mine) == budget
                    worst = max(edge[t] for t in theirs - mine) - min(edge[t] for t in mine - theirs)
                    assert 0 <= worst <= 2e-3, worst
                weight = dict((t, x) for t, x in rows)
                state[b, h] = [[t, weight[t]] for t in positions[0, b, h, :budget].tolist()]
            else:
                assert (positions[0, b, h, :n] == -1).all() or n <= budget
            got_s = scores[0, b, h, : len(state[b, h])].double().cpu().numpy()
            # the prompt's lse comes from rounded weights (2^-8 of each weight), the steps' from fp32 sums
            assert (np.abs(got_s - [x for _, x in state[b, h]]) <= 2.0 ** -8 * got_s + 1e-3).all()
        for _ in range(grow):
            n = lens.tolist()
            append([(b, n[b], int(total[b])) for b in range(B)])
            lens += 1
            q = torch.randn((B, 32, 128), generator=gen).to(torch.bfloat16)
            out, step_lse = ops.decode_attention_scored(q.cuda(), cache, table, lens, scores[0],
                                                        lse=torch.empty((B, 32), device="cuda"))
            for b in range(B):
                for h in range(8):
                    rows = state[b, h]
                    rows.append([int(total[b]), 0.0])
                    toks = [t for t, _ in rows]
                    kk, vv = k[b, toks, h: h + 1].double().numpy(), v[b, toks, h: h + 1].double().numpy()
                    qq = q[b: b + 1, 4 * h: 4 * h + 4].double().numpy()
                    want, want_lse, w, tol = ow.attend(qq, kk, vv, np.ones((1, len(toks)), bool), SCALE, True)
                    assert (np.abs(out[b, 4 * h: 4 * h + 4].double().cpu().numpy() - want[0]) <= tol[0] + 2.0 ** -11 * 5).all()
                    assert np.abs(step_lse[b, 4 * h: 4 * h + 4].cpu().numpy() - want_lse[0]).max() <= 1e-4
                    for row, x in zip(rows, w.sum((0, 1))):
                        row[1] += x
            total += 1
