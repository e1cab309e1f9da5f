"""The cache in 4 bits on the GPU: rows in and out byte by byte, attention over them against the float64 oracle."""
import numpy as np
import pytest
import torch

from oracle import int4 as oi

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5
PAGE_BYTES = 20480


def _bf(seed, shape, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(torch.bfloat16)


def _edge_rows(seed):
    """Rows whose groups are of every kind: constant, zero, negative zeros, tiny, huge, one loud dim, ties, not finite."""
    x = _bf(seed, (24, 8, 128)).float()
    x[0] = 0
    x[1] = -2.5
    x[2, :, ::2], x[2, :, 1::2] = 0.0, -0.0
    x[3] *= 1e-38
    x[4] *= 2e-40
    x[5] *= 1e37
    x[6, :, 17] = 300.0
    x[7] = torch.arange(128).float() % 16                    # codes as they are
    x[8] = (torch.arange(128) % 31).float() / 2              # halves of a step
    x[9, 0, 3], x[9, 1, 40], x[9, 2, 127] = float("inf"), float("nan"), float("-inf")
    x[10, :, 0], x[10, :, 1] = 3e38, -3e38
    x[11] = 1000 + _bf(seed + 1, (8, 128)).float()
    return x.to(torch.bfloat16)


@pytest.mark.parametrize("T", [1, 3, 24, 257])
def test_rows_in_and_out(T):
    """Bytes as the oracle writes them, values as it reads them; skipped tokens and other slots as they were."""
    from abridgekv_amd import ops
    k, v = _bf(1, (T, 8, 128), 2.0), _bf(2, (T, 8, 128))
    k[:24], v[:24] = _edge_rows(3)[:T], _edge_rows(5)[:T]
    pool = -(-T // 16) + 3
    cache = torch.randint(0, 256, ops.kv_cache_int4_shape(pool), dtype=torch.uint8, generator=torch.Generator().manual_seed(7))
    before = cache.clone().numpy()
    slots = torch.from_numpy(np.random.default_rng(T).permutation(16 * pool)[:T].astype(np.int64))
    skip = [i for i in range(T) if i % 7 == 3]
    slots[skip] = -1
    if T > 30:
        slots[28] = 16 * pool                                # past the cache
        skip.append(28)
    dev = cache.cuda()
    ops.kv_append_int4(k.cuda(), v.cuda(), slots.cuda(), dev)
    want = before.reshape(pool, 2, 16, 640).copy()
    for t in range(T):
        if t not in skip:
            s = int(slots[t])
            want[s // 16, 0, s % 16] = oi.quantise(k[t: t + 1].float().numpy())[0]
            want[s // 16, 1, s % 16] = oi.quantise(v[t: t + 1].float().numpy())[0]
    assert np.array_equal(dev.cpu().numpy(), want)
    for dtype, tol in ((torch.float32, 2.0 ** -24), (torch.bfloat16, 2.0 ** -8)):
        got = ops.kv_read_int4(dev, slots.cuda(), dtype)
        for half, g in enumerate(got):
            assert g.dtype == dtype and g.shape == (T, 8, 128)
            for t in range(T):
                if t in skip:
                    assert not g[t].any()
                    continue
                s = int(slots[t])
                val = oi.values(want[s // 16, half, s % 16][None])[0]
                have = g[t].double().cpu().numpy()
                fin = np.isfinite(val) & (np.abs(val) < 3e38)
                assert np.array_equal(np.isnan(val), np.isnan(have) & ~np.isfinite(val))
                # a product of 8 and 4 bits is exact in fp32: one rounding of the sum (tiny values: the smallest subnormal)
                assert (np.abs(have - val)[fin] <= tol * 1.01 * np.abs(val)[fin] + 2e-45 + (dtype == torch.bfloat16) * 1e-40).all()


def test_rows_of_a_fused_projection():
    """Keys and values as slices of one [T, 48 * 128] projection, and heads in another order of memory."""
    from abridgekv_amd import ops
    qkv = _bf(4, (33, 48, 128)).cuda()
    k, v = qkv[:, 32:40], qkv[:, 40:]
    slots = torch.arange(33, device="cuda") + 7
    a, b = (torch.zeros(ops.kv_cache_int4_shape(3), dtype=torch.uint8, device="cuda") for _ in range(2))
    ops.kv_append_int4(k, v, slots, a)
    ops.kv_append_int4(k.contiguous(), v.transpose(0, 1).contiguous().transpose(0, 1), slots, b)
    assert torch.equal(a, b) and a.any()


def _paged(lens, seed, extra=5, loud=True):
    """Rows of each sequence (bytes) in a cache of scattered pages; every other byte is arbitrary."""
    rng = np.random.default_rng(seed)
    need = [-(-n // 16) for n in lens]
    pool = sum(need) + extra
    pages = rng.permutation(pool)[: sum(need)]
    table = rng.integers(-5, pool + 9, (len(lens), max(1, max(need)))).astype(np.int32)
    cache = rng.integers(0, 256, (pool, 2, 16, 640)).astype(np.uint8)
    ks, vs, at = [], [], 0
    for b, n in enumerate(lens):
        table[b, : need[b]] = pages[at: at + need[b]]
        at += need[b]
        k, v = (_bf(seed * 1000 + 2 * b + i, (n, 8, 128)).float() for i in (0, 1))
        if loud:
            k[:, :, 5] += 6.0                                # a dim that is loud in every row
            v += 0.5
        ks.append(oi.quantise(oi.bf16(k.numpy())))
        vs.append(oi.quantise(oi.bf16(v.numpy())))
        pos = np.arange(n)
        cache[table[b, pos // 16], 0, pos % 16] = ks[-1]
        cache[table[b, pos // 16], 1, pos % 16] = vs[-1]
    q = _bf(seed + 77, (len(lens), 32, 128))
    return q, ks, vs, torch.from_numpy(cache).cuda(), torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32).cuda()


def _close(out, lse, q, k, v, vis, wide=False):
    want, want_lse, tol, ltol = oi.attend(q.double().numpy(), k, v, vis, SCALE, wide)
    err = np.abs(out.double().cpu().numpy() - want)
    assert (err <= tol).all(), (err - tol).max()
    if lse is not None:
        some = vis.any(1)
        got = lse.double().cpu().numpy()
        assert (np.abs(got[some] - want_lse[some]) <= ltol[some]).all() and (got[~some] == -np.inf).all()
    assert not out.cpu()[torch.from_numpy(~vis.any(1))].any()


LENS = [0, 1, 15, 16, 17, 33, 100, 511, 513, 1300]


@pytest.mark.parametrize("split_pages", [0, 2, 8, 64, None])
def test_decode(split_pages):
    from abridgekv_amd import ops
    q, k, v, cache, table, sl = _paged(LENS, 11)
    lse = torch.empty((len(LENS), 32), device="cuda")
    out, got = ops.decode_attention_int4(q.cuda(), cache, table, sl, lse=lse, split_pages=split_pages)
    assert got is lse
    for b, n in enumerate(LENS):
        _close(out[b: b + 1], lse[b: b + 1], q[b: b + 1], k[b], v[b], np.ones((1, n), bool))


@pytest.mark.parametrize("lens", [[1], [32], [33], [5000], [9000, 1], [0] * 5, [7] * 300, [0, 2100, 0, 0, 31, 4097, 64, 1, 0], "many", "long"])
def test_decode_in_shares(lens):
    """Equal shares against splits: shares that end inside sequences, at their ends, that hold many of them, empty ones; few
    sequences, 512, and enough rows for shares of more than 64 pages."""
    from abridgekv_amd import ops
    if lens == "many":
        lens = np.random.default_rng(5).integers(0, 400, 512).tolist()
    if lens == "long":
        lens = [33000 + 1000 * i for i in range(40)]
    B, W = len(lens), max(1, -(-max(lens) // 16))
    gen = torch.Generator(device="cuda").manual_seed(B)
    k, v = (torch.randn((16 * 500, 8, 128), device="cuda", generator=gen).to(torch.bfloat16) for _ in range(2))
    cache = torch.zeros(ops.kv_cache_int4_shape(500), dtype=torch.uint8, device="cuda")
    ops.kv_append_int4(k, v, torch.arange(16 * 500, device="cuda"), cache)
    table = torch.randint(0, 500, (B, W), device="cuda", dtype=torch.int32, generator=gen)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn((B, 32, 128), device="cuda", generator=gen).to(torch.bfloat16)
    la, lb = (torch.full((B, 32), 3.0, device="cuda") for _ in range(2))
    a, _ = ops.decode_attention_int4(q, cache, table, sl, lse=la, split_pages=0)
    b, _ = ops.decode_attention_int4(q, cache, table, sl, lse=lb, split_pages=64)
    some = sl > 0
    assert not a[~some].any() and (la[~some] == -np.inf).all()
    # each has a weight times a step rounded to bf16 (2^-8, errors that part ways where the running maxima differ) of values
    # within 8 steps of the middle, its output rounded (2^-8), parts in fp16 (2^-11 of the largest value): twice their sum
    step, largest = 0.8, 6.0                                 # of rows of normal numbers: (max - min) / 15, and of any value
    size = 8 * step + a.float().abs() + largest * 2.0 ** -3
    assert ((a.float() - b.float()).abs() <= 2 * 2.0 ** -8 * size).all()
    assert torch.allclose(la[some], lb[some], rtol=1e-5, atol=1e-4)
    c, _ = ops.decode_attention_int4(q, cache, table, sl, split_pages=0)
    assert torch.equal(a, c)
    if B > 40:
        for i in (0, B // 2, B - 1):
            n, t = lens[i], table[i].long().cpu().numpy()
            rows = cache.cpu().numpy()[t[np.arange(n) // 16], :, np.arange(n) % 16] if n else np.zeros((0, 2, 640), np.uint8)
            _close(a[i: i + 1], la[i: i + 1], q[i: i + 1].cpu(), np.ascontiguousarray(rows[:, 0]), np.ascontiguousarray(rows[:, 1]),
                   np.ones((1, n), bool))


def test_shares_in_a_graph():
    """A captured decode in shares follows lengths that change between replays, through the custom op and its workspace, beside
    eager calls with a workspace of their own."""
    from abridgekv_amd import ops, torch_ops  # noqa: F401
    B, W = 48, 200
    gen = torch.Generator(device="cuda").manual_seed(3)
    cache = torch.zeros(ops.kv_cache_int4_shape(300), dtype=torch.uint8, device="cuda")
    k, v = (torch.randn((16 * 300, 8, 128), device="cuda", generator=gen).to(torch.bfloat16) for _ in range(2))
    ops.kv_append_int4(k, v, torch.arange(16 * 300, device="cuda"), cache)
    table = torch.randint(0, 300, (B, W), device="cuda", dtype=torch.int32, generator=gen)
    q = torch.randn((B, 32, 128), device="cuda", generator=gen).to(torch.bfloat16)
    sl = torch.randint(0, 16 * W + 1, (B,), device="cuda", dtype=torch.int32, generator=gen)
    assert ops.int4_split_pages(B, W) == 0
    out, lse = torch.empty_like(q), torch.empty((B, 32), device="cuda")
    ws = ops.decode_int4_workspace(B, W, device="cuda")
    step = lambda: torch.ops.abridgekv.decode_attn_int4(q, cache, table, sl, SCALE, W, 0, out, lse, ws)      # noqa: E731
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        sl.copy_(torch.randint(0, (16 * W, 40)[i % 2] + 1, (B,), device="cuda", dtype=torch.int32, generator=gen))
        graph.replay()
        got, got_lse = out.clone(), lse.clone()
        want_lse = torch.empty_like(lse)
        want, _ = ops.decode_attention_int4(q, cache, table, sl, SCALE, lse=want_lse)
        assert torch.equal(got, want) and torch.equal(got_lse, want_lse)


def test_decode_bounds_and_views():
    """Lengths past max_pages are cut, queries and outputs are slices, extra table rows and lengths stay unread."""
    from abridgekv_amd import ops
    lens = [90, 300, 5]
    q, k, v, cache, table, sl = _paged(lens, 12)
    qs = torch.zeros((3, 48, 128), dtype=torch.bfloat16, device="cuda")
    qs[:, 8:40] = q.cuda()
    outs = torch.full((3, 40, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.decode_attention_int4(qs[:2, 8:40], cache, table, sl, max_pages=4, out=outs[:2, 4:36])
    for b in range(2):
        n = min(lens[b], 64)
        _close(outs[b: b + 1, 4:36], None, q[b: b + 1], k[b][:n], v[b][:n], np.ones((1, n), bool))
    assert (outs[2] == 7).all() and (outs[:, :4] == 7).all() and (outs[:, 36:] == 7).all()


def test_decode_scores_far_apart():
    """One row that outweighs the rest, first, last or in the middle of a split, and scores of hundreds."""
    from abridgekv_amd import ops
    lens = [200, 200, 200]
    q, k, v, cache, table, sl = _paged(lens, 13, loud=False)
    for b, row in enumerate((0, 150, 199)):
        big = oi.quantise(oi.bf16(40 * q[b].float().view(8, 4, 128).mean(1).numpy()[None]))
        k[b][row] = big[0]
        cache[table[b, row // 16], 0, row % 16] = torch.from_numpy(big[0]).cuda()
    lse = torch.empty((3, 32), device="cuda")
    for split in (4, 64):
        out, _ = ops.decode_attention_int4(q.cuda(), cache, table, sl, lse=lse, split_pages=split)
        for b in range(3):
            _close(out[b: b + 1], lse[b: b + 1], q[b: b + 1], k[b], v[b], np.ones((1, 200), bool))


def test_decode_row_that_is_not_finite():
    """A NaN group reaches its sequence and KV head and no other."""
    from abridgekv_amd import ops
    q, k, v, cache, table, sl = _paged([70, 70], 14)
    good, _ = ops.decode_attention_int4(q.cuda(), cache, table, sl)
    pairs = cache.view(-1, 2, 16, 640)[int(table[0, 1]), 1, 3, 512 + 16 * 2: 512 + 16 * 2 + 2]      # value row 19, head 2, group 0
    pairs.copy_(torch.tensor([0xC0, 0x7F], dtype=torch.uint8))
    out, _ = ops.decode_attention_int4(q.cuda(), cache, table, sl)
    assert torch.isnan(out[0, 8:12, :32]).all()
    rest = torch.ones_like(out, dtype=torch.bool)
    rest[0, 8:12] = False
    assert torch.equal(out[rest], good[rest])


def test_offsets_past_32_bits():
    """Pages beyond 4 GiB of cache."""
    from abridgekv_amd import ops
    pool = (1 << 32) // PAGE_BYTES + 40
    cache = torch.zeros(ops.kv_cache_int4_shape(pool), dtype=torch.uint8, device="cuda")
    n = 100
    k, v, q = _bf(1, (n, 8, 128)), _bf(2, (n, 8, 128)), _bf(3, (1, 32, 128))
    table = torch.arange(pool - 8, pool, dtype=torch.int32, device="cuda")[None]
    slots = (pool - 8) * 16 + torch.arange(n, device="cuda")
    ops.kv_append_int4(k.cuda(), v.cuda(), slots, cache)
    kr, vr = oi.quantise(k.float().numpy()), oi.quantise(v.float().numpy())
    got = ops.kv_read_int4(cache, slots)[0].double().cpu().numpy()
    assert np.abs(got - oi.values(kr)).max() <= 2.0 ** -22
    sl = torch.tensor([n], dtype=torch.int32, device="cuda")
    out, _ = ops.decode_attention_int4(q.cuda(), cache, table, sl)
    _close(out, None, q, kr, vr, np.ones((1, n), bool))
    out, _ = ops.paged_prefill_attention_int4(q.cuda(), cache, table, [0, 1], [n - 1], [n], True)
    _close(out, None, q, kr, vr, np.ones((1, n), bool), wide=True)


# requests: (queries, rows before them, key limit or None: causal, excluded range or None)
BATCHES = {
    "one token": [(1, 0, None, None)],
    "short": [(3, 70, None, None), (17, 0, None, None)],
    "tile edges": [(64, 0, None, None), (65, 1, None, None), (63, 64, None, None)],
    "code step": [(128, 500, 500 + 32, None)],
    "tail hidden": [(40, 200, 240, (180, 200)), (1, 30, None, None)],
    "mixed": [(100, 900, None, None), (130, 0, None, None), (64, 300, 300 + 16, (290, 300)), (1, 1299, None, None)],
    "nothing to see": [(5, 0, 0, None), (7, 9, None, None)],
}


@pytest.mark.parametrize("name", BATCHES)
def test_chunks(name):
    from abridgekv_amd import ops
    reqs = BATCHES[name]
    lens = [past + n for n, past, _, _ in reqs]
    _, k, v, cache, table, _ = _paged(lens, 15)
    starts = np.concatenate([[0], np.cumsum([r[0] for r in reqs])])
    T = int(starts[-1])
    q = _bf(16, (T + 3, 32, 128))
    out = torch.full((T + 3, 32, 128), 5.0, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((T + 3, 32), 5.0, device="cuda")
    limits = [lens[r] if lim is None else lim for r, (_, _, lim, _) in enumerate(reqs)]
    ops.paged_prefill_attention_int4(q.cuda(), cache, table, starts, [r[1] for r in reqs], limits, [r[2] is None for r in reqs],
                                     out=out, lse=lse, excluded=[r[3] for r in reqs])
    assert (out[T:] == 5).all() and (lse[T:] == 5).all()
    for r, (n, past, lim, ex) in enumerate(reqs):
        j = np.arange(lens[r])[None]
        vis = np.repeat(j < limits[r], n, 0) & ((lim is not None) | (j <= past + np.arange(n)[:, None]))
        if ex is not None:
            vis &= (j < ex[0]) | (j >= ex[1])
        sl = slice(starts[r], starts[r + 1])
        _close(out[sl], lse[sl], q[sl], k[r], v[r], vis, wide=True)


RANGES = {                                                   # powers of two of page p's keys and values, of the queries
    "values grow": (lambda p: 0, lambda p: 4 * p, 0),
    "values shrink": (lambda p: 0, lambda p: 60 - 5 * p, 0),
    "values huge and tiny": (lambda p: 0, lambda p: (100, -100)[p % 2], 0),
    "all tiny": (lambda p: -30, lambda p: -60, 30),
    "keys differ by page": (lambda p: (0, -12, -24)[p % 3], lambda p: 0, 0),
    "queries tiny": (lambda p: 24, lambda p: 3, -24),
    "queries huge": (lambda p: -70, lambda p: 0, 70),
}


@pytest.mark.parametrize("name", RANGES)
def test_any_range(name):
    """Magnitudes far outside fp16's, alike in a sequence and changing from page to page: chunks, and single tokens."""
    from abridgekv_amd import ops
    of_k, of_v, of_q = RANGES[name]
    n, nq = 400, 70
    rows = []
    for seed, of in ((31, of_k), (32, of_v)):
        x = _bf(seed, (n, 8, 128)).float()
        x *= torch.tensor([2.0 ** of(i // 16) for i in range(n)])[:, None, None]
        rows.append(oi.quantise(oi.bf16(x.numpy())))
    q = (_bf(33, (nq, 32, 128)).float() * 2.0 ** of_q).to(torch.bfloat16)
    pages = -(-n // 16)
    cache = np.zeros((pages, 2, 16, 640), np.uint8)
    at = np.arange(n)
    for half in (0, 1):
        cache[at // 16, half, at % 16] = rows[half]
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    lse = torch.empty((nq, 32), device="cuda")
    out, _ = ops.paged_prefill_attention_int4(q.cuda(), torch.from_numpy(cache).cuda(), table, [0, nq], [n - nq], [n], True, lse=lse)
    vis = np.arange(n)[None] <= n - nq + np.arange(nq)[:, None]
    _close(out, lse, q, *rows, vis, wide=True)
    sl = torch.tensor([n], dtype=torch.int32, device="cuda")
    for split in (2, 64):
        one, _ = ops.decode_attention_int4(q[-1:].cuda(), torch.from_numpy(cache).cuda(), table, sl, lse=lse[:1], split_pages=split)
        _close(one, lse[:1], q[-1:], *rows, np.ones((1, n), bool))


def test_chunk_row_that_is_not_finite():
    """A NaN group of values reaches the queries that see it, in its dims and KV head, and nothing else of its page."""
    from abridgekv_amd import ops
    _, _, _, cache, table, _ = _paged([300], 34)
    q = _bf(35, (40, 32, 128)).cuda()
    args = (table, [0, 40], [260], [300], True)
    good, _ = ops.paged_prefill_attention_int4(q, cache, *args)
    pairs = cache[int(table[0, 1]), 1, 3, 512 + 16 * 2: 512 + 16 * 2 + 2]        # value row 19, head 2, group 0
    pairs.copy_(torch.tensor([0xC0, 0x7F], dtype=torch.uint8))
    out, _ = ops.paged_prefill_attention_int4(q, cache, *args)
    assert torch.isnan(out[:, 8:12, :32]).all()
    rest = torch.ones_like(out, dtype=torch.bool)
    rest[:, 8:12, :32] = False
    assert torch.equal(out[rest], good[rest])


def test_row_moves():
    """Compaction moves of a 4-bit cache: whole rows of bytes, ordered and independent, one launch and several groups, and the
    staged form."""
    from abridgekv_amd import ops
    rng = np.random.default_rng(2)
    pool, layers = 30, 3
    host = [rng.integers(0, 256, (pool, 2, 16, 640)).astype(np.uint8) for _ in range(layers)]

    def op(src, dst):
        return [src // 16, src % 16, dst // 16, dst % 16]

    ordered = [op(40 + i, 10 + i) for i in range(90)]                   # a run moved down within pages 0 .. 8
    free = [op(160 + i, 320 + i) for i in range(50)]
    want = [h.copy() for h in host]
    for h, w in zip(host, want):
        for a, b, c, d in ordered + free:
            w[c, :, d] = h[a, :, b]
    o = torch.tensor(ordered, dtype=torch.int32, device="cuda")
    f = torch.tensor(free, dtype=torch.int32, device="cuda")
    seg = torch.tensor([0, len(ordered)], dtype=torch.int32, device="cuda")
    none = torch.empty((0, 4), dtype=torch.int32, device="cuda")

    def caches():
        return [torch.from_numpy(h).cuda() for h in host]

    for call in (lambda c: ops.kv_move_mixed(c, o, seg, f),
                 lambda c: ops.kv_move_groups([(c, o, seg, none), (c, none, seg[:1], f)]),
                 lambda c: (ops.kv_move_segments(c, o, seg), ops.kv_copy_staged(c, f))):
        got = caches()
        call(got)
        assert all(np.array_equal(g.cpu().numpy(), w) for g, w in zip(got, want))


def test_capture_and_streams():
    """A step's append and attention on another stream, recorded once and replayed with new rows: as the eager calls."""
    from abridgekv_amd import ops
    lens = [130, 61]
    q, k, v, cache, table, sl = _paged([x + 5 for x in lens], 17)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    qs, ks, vs = _bf(18, (5, 2, 32, 128)).cuda(), _bf(19, (5, 2, 8, 128)).cuda(), _bf(20, (5, 2, 8, 128)).cuda()
    other = cache.clone()
    q1, k1, v1, out = qs[0].clone(), ks[0].clone(), vs[0].clone(), torch.empty_like(qs[0])
    slots = torch.empty(2, dtype=torch.int64, device="cuda")
    ws = ops.decode_int4_workspace(2, table.shape[1], 4, device="cuda")
    n = sl.clone()

    def place(lengths):
        return torch.stack([table[b, int(x) // 16].long() * 16 + int(x) % 16 for b, x in enumerate(lengths.tolist())])

    def step():
        ops.kv_append_int4(k1, v1, slots, other)
        ops.decode_attention_int4(q1, other, table, n, out=out, split_pages=4, workspace=ws)

    side = torch.cuda.Stream()
    slots.copy_(place(n))
    n += 1
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    want_n = sl.clone()
    for i in range(5):
        slots.copy_(place(want_n))
        want_n += 1
        n.copy_(want_n)
        for a, b in ((q1, qs), (k1, ks), (v1, vs)):
            a.copy_(b[i])
        graph.replay()
        torch.cuda.synchronize()
        ops.kv_append_int4(ks[i], vs[i], slots, cache)
        want, _ = ops.decode_attention_int4(qs[i], cache, table, want_n, split_pages=4)
        assert torch.equal(out, want), i
    assert torch.equal(cache, other)
