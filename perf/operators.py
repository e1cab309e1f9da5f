"""The performance cases of the operators that bound a context: attention with a sliding window and sinks, attention
weights accumulated per cached row, and eviction of cached rows by them.

A case is a dict of plain values; ``kind`` names the call:

  prompt   attention under the window over whole prompts (``ops.window_attention``), bf16 or fp32
  train    the same through the attention function the models register, with the gradients of q, k and v
  chunk    prompt chunks of several requests over the paged cache (``ops.paged_prefill_attention_window``)
  token    one new token per sequence over the paged cache (``ops.decode_attention_window``)
  weigh    a decode step that adds its attention weights to the rows' scores (``ops.decode_attention_scored``)
  observe  the weights of a prompt's queries, added to the rows' scores (``ops.paged_prefill_scores``)
  evict    rows leave the cache by score (``ops.kv_evict``)

Geometry: 32 query heads, 8 KV heads, head size 128, pages of 16 rows. Query row i sees key row j when j <= i and
(i - j < window or j < sinks). Lengths inside a batch are spread over the case's range in an order fixed by the case,
so that every seed has the same amount of work.
"""
from __future__ import annotations

import math
import types

import numpy as np
import torch

own = False

HQ, HKV, D, PAGE = 32, 8, 128, 16
G = HQ // HKV
SCALE = 1.0 / math.sqrt(D)


def listed():
    return [
        # evaluation of two documents under a window, one of them shorter (padded batch)
        {"name": "prompt_8192", "kind": "prompt", "dtype": "bf16", "B": 2, "S": 8192, "len_min": 5000, "window": 1024,
         "sinks": 4},
        # the same attention in float32, as a parity run of a model in float32 uses it
        {"name": "prompt_f32", "kind": "prompt", "dtype": "f32", "B": 1, "S": 1500, "len_min": 1500, "window": 512,
         "sinks": 4},
        # a small ragged training batch with an odd window and a long run of sinks
        {"name": "train_777", "kind": "train", "dtype": "bf16", "B": 3, "S": 777, "len_min": 300, "window": 129,
         "sinks": 17},
        # a training step's attention
        {"name": "train_4096", "kind": "train", "dtype": "bf16", "B": 2, "S": 4096, "len_min": 4096, "window": 512,
         "sinks": 4},
        # a serving step's prompt chunks, some far into their prompts
        {"name": "chunk_4", "kind": "chunk", "dtype": "bf16", "R": 4, "chunk_min": 300, "chunk_max": 512,
         "past_min": 0, "past_max": 8000, "window": 1024, "sinks": 4},
        # one request decoding alone, far past its window (latency bound)
        {"name": "token_1", "kind": "token", "dtype": "bf16", "B": 1, "rows_min": 32000, "rows_max": 32000,
         "window": 1024, "sinks": 4},
        # a batch of 64 under a wide window, some sequences still inside it
        {"name": "token_64", "kind": "token", "dtype": "bf16", "B": 64, "rows_min": 2000, "rows_max": 32000,
         "window": 4096, "sinks": 4},
        # one request decoding alone with a budget of 2048 rows
        {"name": "weigh_1", "kind": "weigh", "dtype": "bf16", "B": 1, "rows_min": 2100, "rows_max": 2100},
        # a batch of 64 with a budget of 2048 rows, up to 512 rows since the last eviction
        {"name": "weigh_64", "kind": "weigh", "dtype": "bf16", "B": 64, "rows_min": 2049, "rows_max": 2560},
        # two prompts whose queries weigh every row
        {"name": "observe_2", "kind": "observe", "dtype": "bf16", "R": 2, "chunk_min": 1500, "chunk_max": 2048,
         "past_min": 0, "past_max": 2048},
        # one sequence of one KV-cache group of six layers passes its budget
        {"name": "evict_1", "kind": "evict", "layers": 6, "B": 1, "rows_min": 2560, "rows_max": 2560, "budget": 2048,
         "sinks": 4, "recent": 256},
        # a batch of 64 after 400 to 512 steps
        {"name": "evict_64", "kind": "evict", "layers": 6, "B": 64, "rows_min": 2448, "rows_max": 2560,
         "budget": 2048, "sinks": 4, "recent": 256},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "train", "train", "chunk", "token", "token", "weigh", "weigh", "observe",
                       "evict", "evict"])
    if kind in ("prompt", "train"):
        f32 = kind == "prompt" and rng.random() < 0.3
        S = _log(rng, 1, 1500 if f32 else 8192 if kind == "prompt" else 4096)
        B = rng.randint(1, max(1, min(4, 8192 // S)))
        return {"kind": kind, "dtype": "f32" if f32 else "bf16", "B": B, "S": S, "len_min": rng.randint(0, S),
                "window": _log(rng, 1, 1024), "sinks": rng.choice([0, 1, 4, 4, 16, rng.randint(0, 200)])}
    if kind in ("chunk", "observe"):
        c0, c1 = sorted((_log(rng, 1, 512 if kind == "chunk" else 1500), _log(rng, 2, 512 if kind == "chunk" else 1500)))
        case = {"kind": kind, "dtype": "bf16", "R": rng.randint(1, 4 if kind == "chunk" else 2), "chunk_min": c0,
                "chunk_max": c1, "past_min": 0, "past_max": rng.choice([0, _log(rng, 1, 2000)])}
        if kind == "chunk":
            case.update(past_max=rng.choice([0, _log(rng, 1, 8000)]), window=_log(rng, 1, 1024),
                        sinks=rng.choice([0, 4, 4, rng.randint(0, 200)]))
        return case
    if kind in ("token", "weigh"):
        B = _log(rng, 1, 64)
        lo, hi = sorted((_log(rng, 1, 32000 if kind == "token" else 2560), _log(rng, 1, 32000 if kind == "token" else 2560)))
        case = {"kind": kind, "dtype": "bf16", "B": B, "rows_min": lo, "rows_max": hi}
        if kind == "token":
            case.update(window=_log(rng, 1, 4096), sinks=rng.choice([0, 4, 4, rng.randint(0, 200)]))
        return case
    budget = _log(rng, 16, 2048)
    recent = rng.randint(0, budget // 2)
    lo, hi = sorted((rng.randint(max(1, budget // 2), budget + 512), rng.randint(budget, budget + 512)))
    return {"kind": kind, "layers": rng.randint(1, 6), "B": _log(rng, 1, 64), "rows_min": lo, "rows_max": hi,
            "budget": budget, "sinks": rng.randint(0, min(16, budget - recent)), "recent": recent}


# -- sizes and inputs ------------------------------------------------------------------------------------------------
def _spread(n, lo, hi, salt):
    """n lengths over [lo, hi], both ends among them (n > 1), in an order fixed by the sizes."""
    v = np.round(np.linspace(lo, hi, n)).astype(np.int64) if n > 1 else np.array([hi], np.int64)
    return np.random.RandomState(17 * n + salt).permutation(v)


def _lengths(case):
    kind = case["kind"]
    if kind in ("prompt", "train"):
        return _spread(case["B"], case["len_min"], case["S"], 1)
    return _spread(case["B"], case["rows_min"], case["rows_max"], 2)


def _chunks(case):
    """Chunk lengths and the rows before each."""
    return (_spread(case["R"], case["chunk_min"], case["chunk_max"], 3),
            _spread(case["R"], case["past_min"], case["past_max"], 4))


def _randn(gen, shape, dtype=torch.bfloat16):
    x = torch.empty(shape, dtype=dtype, device="cuda")
    return x.normal_(generator=gen)


def _paged(gen, lens, spare=4):
    """A page table [B, W] int32 for sequences of these lengths over scattered pages, and the pages of the pool."""
    need = -(-np.asarray(lens) // PAGE)
    pool = int(need.sum()) + spare
    ids = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32).cpu().numpy()
    tab = np.zeros((len(need), max(1, int(need.max()))), np.int32)
    at = 0
    for b, n in enumerate(need):
        tab[b, :n] = ids[at: at + n]
        at += n
    return torch.from_numpy(tab).cuda(), pool


def _spans(window, sinks, lens):
    """Rows the last token of sequences of these lengths sees."""
    start = np.maximum(lens - window, 0)
    return np.minimum(sinks, start) + lens - start


def prepare(case, seed):
    s = types.SimpleNamespace(case=case)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 1000003 + 7)
    kind = case["kind"]
    dt = torch.float32 if case.get("dtype") == "f32" else torch.bfloat16
    if kind in ("prompt", "train"):
        B, S = case["B"], case["S"]
        s.q, s.k, s.v = (_randn(gen, (B, S, h, D), dt) for h in (HQ, HKV, HKV))
        s.lens = torch.from_numpy(_lengths(case).astype(np.int32)).cuda()
        if kind == "train":
            s.dout = _randn(gen, (B, S, HQ, D), dt)
            s.q, s.k, s.v = (t.transpose(1, 2).requires_grad_(True) for t in (s.q, s.k, s.v))   # as a model hands them
            s.module = types.SimpleNamespace(layer_idx=0)
        return s
    if kind in ("chunk", "observe"):
        n, past = _chunks(case)
        s.table, pool = _paged(gen, n + past)
        s.cache = _randn(gen, (pool, 2, PAGE, HKV, D))
        s.q = _randn(gen, (int(n.sum()), HQ, D))
        s.q_start, s.kv_start = np.concatenate([[0], np.cumsum(n)]), past
        if kind == "observe":                                # the chunk's attention ran before and left its lse
            s.lse = torch.cat([_attend64(s, r)[1] for r in range(case["R"])]).float()
            s.scores = torch.rand((case["R"], HKV, s.table.shape[1] * PAGE), generator=gen, device="cuda") * 4
        return s
    lens = _lengths(case)
    B = case["B"]
    s.table, pool = _paged(gen, lens)
    s.lens = torch.from_numpy(lens.astype(np.int32)).cuda()
    M = s.table.shape[1] * PAGE
    if kind == "evict":
        L = case["layers"]
        s.caches = [_randn(gen, (pool, 2, PAGE, HKV, D)) for _ in range(L)]
        # weights summed over many steps: a few rows hold most of them
        s.scores = torch.empty((L, B, HKV, M), device="cuda").log_normal_(0.0, 2.0, generator=gen)
        s.positions = torch.full((L, B, HKV, M), -1, dtype=torch.int32, device="cuda")
        s.grown = torch.from_numpy(np.maximum(lens - case["budget"], 0).astype(np.int32)).cuda()
        s.tokens = s.lens - s.grown                          # run() adds the rows appended since the last call
        return s
    s.cache = _randn(gen, (pool, 2, PAGE, HKV, D))
    s.q = _randn(gen, (B, HQ, D))
    if kind == "weigh":
        s.scores = torch.rand((B, HKV, M), generator=gen, device="cuda") * 4
    return s


# -- one pass --------------------------------------------------------------------------------------------------------
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from abridgekv_amd import ops
    from abridgekv_amd.compress_forward import WindowMask, masked_attention_forward

    case = s.case
    kind = case["kind"]
    if kind == "prompt":
        return {"out": ops.window_attention(s.q, s.k, s.v, case["window"], case["sinks"], seq_lens=s.lens, scale=SCALE)[0]}
    if kind == "train":
        mask = WindowMask(case["window"], case["sinks"], s.lens)
        out, _ = masked_attention_forward(s.module, s.q, s.k, s.v, mask, scaling=SCALE)
        dq, dk, dv = torch.autograd.grad(out, (s.q, s.k, s.v), s.dout)
        return {"out": out, "dq": dq, "dk": dk, "dv": dv}
    if kind == "chunk":
        return {"out": ops.paged_prefill_attention_window(s.q, s.cache, s.table, s.q_start, s.kv_start, case["window"],
                                                          case["sinks"], scale=SCALE)[0]}
    if kind == "token":
        lse = torch.empty((case["B"], HQ), device="cuda")
        out, _ = ops.decode_attention_window(s.q, s.cache, s.table, s.lens, case["window"], case["sinks"], SCALE, lse=lse)
        return {"out": out, "lse": lse}
    if kind == "weigh":
        lse = torch.empty((case["B"], HQ), device="cuda")
        out, _ = ops.decode_attention_scored(s.q, s.cache, s.table, s.lens, s.scores, SCALE, lse=lse)
        return {"out": out, "lse": lse, "scores": s.scores}
    if kind == "observe":
        ops.paged_prefill_scores(s.q, s.cache, s.table, s.q_start, s.kv_start, s.lse, s.scores, scale=SCALE)
        return {"scores": s.scores}
    s.tokens += s.grown
    lens = ops.kv_evict(s.caches, s.table, s.lens, s.scores, s.positions, s.tokens, case["budget"], case["sinks"],
                        case["recent"])
    return {"caches": s.caches, "scores": s.scores, "positions": s.positions, "lens": lens}


def _softmax(sc, vis):
    """Weights and lse of scores sc [..., keys] where vis holds; rows that see nothing have weights 0 and lse -inf."""
    sc = sc.masked_fill_(~vis, -math.inf)
    m = sc.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = sc.sub_(m).exp_()
    z = p.sum(-1, keepdim=True)
    return p.div_(torch.where(z == 0, 1.0, z)), (torch.log(z) + m)[..., 0]


def _grouped(x):
    """[B, S, 32, D] -> [B, 8, 4 S, D] float32, the query heads of a KV head one after the other."""
    B, S = x.shape[:2]
    return x.float().view(B, S, HKV, G, D).permute(0, 2, 3, 1, 4).reshape(B, HKV, G * S, D)


def _ungrouped(x, S):
    return x.view(x.shape[0], HKV, G, S, D).permute(0, 3, 1, 2, 4).reshape(x.shape[0], S, HQ, D)


def _dense_plain(q, k, v, lens, window, sinks, dout=None):
    """q, dout [B, S, 32, D], k, v [B, S, 8, D]: out, and the gradients where dout is given (float32)."""
    S = q.shape[1]
    i = torch.arange(S, device="cuda")
    vis = (i[None] <= i[:, None]) & ((i[:, None] - i[None] < window) | (i[None] < sinks))
    inside = i[None] < lens[:, None]
    vis = vis[None] & inside[:, None] & inside[:, :, None]                          # [B, S, S]
    vis = vis[:, None].repeat(1, 1, G, 1)                                           # [B, 1, 4 S, S]
    qg, kt, vg = _grouped(q), k.float().permute(0, 2, 3, 1).contiguous(), v.float().permute(0, 2, 1, 3).contiguous()
    p, _ = _softmax(torch.matmul(qg, kt).mul_(SCALE), vis)
    out = torch.matmul(p, vg)
    if dout is None:
        return _ungrouped(out, S)
    g = torch.where(inside[:, None, :, None].repeat(1, 1, G, 1), _grouped(dout), 0.0)
    ds = torch.matmul(g, vg.transpose(2, 3).contiguous()).sub_((g * out).sum(-1, keepdim=True)).mul_(p)
    dq = torch.matmul(ds, kt.transpose(2, 3).contiguous()) * SCALE
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), qg) * SCALE
    dv = torch.matmul(p.transpose(2, 3).contiguous(), g)
    return _ungrouped(out, S), _ungrouped(dq, S).transpose(1, 2), dk, dv


def _rows(cache, table, rows):
    """K and V [B, 8, n, D] float32 of slots rows [B, n] (clamped into the table)."""
    rows = rows.clamp(0, table.shape[1] * PAGE - 1)
    kv = cache[torch.gather(table.long(), 1, rows // PAGE), :, rows % PAGE].float()   # [B, n, 2, 8, D]
    return kv[:, :, 0].transpose(1, 2).contiguous(), kv[:, :, 1].transpose(1, 2).contiguous()


def _token_plain(q, cache, table, rows, vis):
    """One token per sequence over the slots rows [B, n] where vis [B, n]: out, lse and the weights [B, 8, 4, n]."""
    k, v = _rows(cache, table, rows)
    p, lse = _softmax(torch.matmul(q.float().view(-1, HKV, G, D), k.transpose(2, 3).contiguous()).mul_(SCALE),
                      vis[:, None, None])
    return torch.matmul(p, v).reshape(-1, HQ, D), lse.reshape(-1, HQ), p


def _chunk_parts(s):
    """A chunk batch padded to its longest request: queries [R, n, 32, D], K and V [R, 8, m, D] float32, the queries'
    positions [R, n], the key slots [m] and which queries are real [R, n]."""
    starts = torch.as_tensor(s.q_start, device="cuda")
    past = torch.as_tensor(s.kv_start, device="cuda")
    lens = starts[1:] - starts[:-1]
    i = torch.arange(int(np.diff(s.q_start).max()), device="cuda")
    real = i[None] < lens[:, None]
    tok = (starts[:-1, None] + i[None]).clamp(max=s.q.shape[0] - 1)
    keys = torch.arange(s.table.shape[1] * PAGE, device="cuda")
    k, v = _rows(s.cache, s.table, keys[None].expand(len(lens), -1))
    return s.q[tok], k, v, past[:, None] + i[None], keys, real, tok


def _run_plain(s):
    case = s.case
    kind = case["kind"]
    if kind == "prompt":
        return {"out": _dense_plain(s.q, s.k, s.v, s.lens, case["window"], case["sinks"]).to(s.q.dtype)}
    if kind == "train":
        q, k, v = (t.detach().transpose(1, 2) for t in (s.q, s.k, s.v))
        got = _dense_plain(q, k, v, s.lens, case["window"], case["sinks"], s.dout)
        return dict(zip(("out", "dq", "dk", "dv"), (t.to(s.q.dtype) for t in got)))
    if kind == "token":
        window, sinks = case["window"], case["sinks"]
        start = (s.lens.long() - window).clamp(min=0)
        first = torch.arange(sinks, device="cuda")[None].expand(case["B"], -1)
        late = start[:, None] + torch.arange(window, device="cuda")[None]
        vis = torch.cat([first < start[:, None], late < s.lens[:, None]], 1)
        out, lse, _ = _token_plain(s.q, s.cache, s.table, torch.cat([first, late], 1), vis)
        return {"out": out.to(s.q.dtype), "lse": lse}
    if kind == "weigh":
        rows = torch.arange(s.scores.shape[2], device="cuda")[None].expand(case["B"], -1)
        out, lse, p = _token_plain(s.q, s.cache, s.table, rows, rows < s.lens[:, None])
        s.scores += p.sum(2)
        return {"out": out.to(s.q.dtype), "lse": lse, "scores": s.scores}
    if kind in ("chunk", "observe"):
        q, k, v, pos, keys, real, tok = _chunk_parts(s)
        n = q.shape[1]
        sc = torch.matmul(_grouped(q), k.transpose(2, 3).contiguous()).mul_(SCALE)              # [R, 8, 4 n, m]
        vis = (keys <= pos[..., None]) & real[..., None]                                        # [R, n, m]
        if kind == "chunk":
            vis = vis & ((pos[..., None] - keys < case["window"]) | (keys < case["sinks"]))
            out = _ungrouped(torch.matmul(_softmax(sc, vis[:, None].repeat(1, 1, G, 1))[0], v), n)
            return {"out": out[real].to(s.q.dtype)}
        lse = s.lse[tok].view(-1, n, HKV, G).permute(0, 2, 3, 1).reshape(-1, HKV, G * n, 1)
        p = sc.sub_(lse).exp_().masked_fill_(~vis[:, None].repeat(1, 1, G, 1), 0.0)
        s.scores += p.sum(2)
        return {"scores": s.scores}
    s.tokens += s.grown
    lens = _evict_plain(s, case["budget"], case["sinks"], case["recent"])
    return {"caches": s.caches, "scores": s.scores, "positions": s.positions, "lens": lens}


def _evict_plain(s, budget, sinks, recent):
    L, B, _, M = s.scores.shape
    slot = torch.arange(M, device="cuda")
    n = s.lens.long()
    m = n.clamp(max=budget)
    over, n4, m4 = (n > budget).view(B, 1, 1), n.view(B, 1, 1), m.view(B, 1, 1)
    tokens = s.tokens.long().view(B, 1, 1)
    pos = torch.where(s.positions < 0, tokens - (n4 - slot), s.positions.long())
    held = (pos < sinks) | (pos >= tokens - recent)
    rank = torch.where(held, math.inf, torch.where(s.scores.isnan(), -math.inf, s.scores)).masked_fill(slot >= n4, -math.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True)[1]
    kept = torch.empty_like(held).scatter_(3, order, (slot < m4).expand(L, B, HKV, M).contiguous())
    hole = ~kept & (slot < m4) & over
    mover = kept & (slot >= m4) & over
    lbh_to, to = hole.view(-1, M).nonzero().unbind(1)                               # ascending slots of each head
    _, frm = mover.view(-1, M).nonzero().unbind(1)
    b, h, layer = lbh_to // HKV % B, lbh_to % HKV, lbh_to // (HKV * B)
    page = lambda x: s.table[b, x // PAGE].long()                                   # noqa: E731
    for i, cache in enumerate(s.caches):
        j = layer == i
        cache[page(to)[j], :, to[j] % PAGE, h[j]] = cache[page(frm)[j], :, frm[j] % PAGE, h[j]]
    flat = s.scores.view(-1, M), pos.view(-1, M)
    gone = over & (slot >= m4) & (slot < n4)
    for state, now, clear in ((s.scores.view(-1, M), flat[0], 0.0), (s.positions.view(-1, M), flat[1], -1)):
        moved = now[lbh_to, frm].to(state.dtype)
        keep = torch.where(over & (slot < n4), now.view(L, B, HKV, M).to(state.dtype), state.view(L, B, HKV, M))
        state.copy_(keep.view(-1, M))
        state[lbh_to, to] = moved
        state.view(L, B, HKV, M).masked_fill_(gone, clear)
    return m.to(torch.int32)


# -- what a pass cannot do without -----------------------------------------------------------------------------------
def _pairs(first, n, window, sinks):
    """Visible pairs of queries first .. first + n - 1 of one sequence."""
    i = np.arange(first, first + n, dtype=np.int64)
    return int(_spans(window, sinks, i + 1).sum())


def work(case):
    kind = case["kind"]
    e = 4 if case.get("dtype") == "f32" else 2
    row = 2 * HKV * D * e                                     # K and V of one row
    if kind in ("prompt", "train"):
        lens = _lengths(case)
        pairs = sum(_pairs(0, int(n), case["window"], case["sinks"]) for n in lens)
        io = int(lens.sum()) * (HQ * D * e + row) + case["B"] * case["S"] * HQ * D * e
        if kind == "prompt":
            return {"bytes": io, "flops": 4 * D * HQ * pairs}
        return {"bytes": io + int(lens.sum()) * HQ * D * e + case["B"] * case["S"] * (HQ * D * e + row),
                "flops": 14 * D * HQ * pairs}
    if kind in ("chunk", "observe"):
        n, past = _chunks(case)
        window, sinks = (case["window"], case["sinks"]) if kind == "chunk" else (1 << 30, 0)
        pairs = sum(_pairs(int(p), int(c), window, sinks) for c, p in zip(n, past))
        reach = np.maximum(past + 1 - window, 0)              # first row of the first query's window
        keys = int((past + n - reach + np.minimum(sinks, reach)).sum())
        T = int(n.sum())
        if kind == "chunk":
            return {"bytes": keys * row + T * HQ * D * 2 * e, "flops": 4 * D * HQ * pairs}
        return {"bytes": keys * (row // 2 + HKV * 8) + T * HQ * (D * e + 4), "flops": 2 * D * HQ * pairs}
    lens = _lengths(case)
    if kind == "token":
        n = int(_spans(case["window"], case["sinks"], lens).sum())
        return {"bytes": n * row + case["B"] * HQ * (2 * D * e + 4), "flops": 4 * D * HQ * n}
    if kind == "weigh":
        n = int(lens.sum())
        return {"bytes": n * (row + HKV * 8) + case["B"] * HQ * (2 * D * e + 4), "flops": 4 * D * HQ * n}
    # every score and position of a sequence over its budget is read; the recent rows leave the slots that go
    over = lens[lens > case["budget"]]
    gone = over - case["budget"]
    moved = int(np.minimum(gone, case["recent"]).sum())
    heads = case["layers"] * HKV
    return {"bytes": max(1, heads * (int(over.sum()) * 8 + int(gone.sum()) * 8 + moved * 2 * (2 * D * 2 + 8))), "flops": 0}


# -- the same results in 64 bits -------------------------------------------------------------------------------------
def _attend64(s, r, window=1 << 30, sinks=0):
    """Out and lse [n, 32, D], [n, 32] float64 of request r's chunk."""
    a, z, past = int(s.q_start[r]), int(s.q_start[r + 1]), int(s.kv_start[r])
    m = past + z - a
    pages = s.cache[s.table[r, : -(-m // PAGE)].long()]
    i = torch.arange(past, m, device="cuda")[:, None]
    j = torch.arange(m, device="cuda")[None]
    hidden = (j > i) | ((i - j >= window) & (j >= sinks))
    out = torch.empty((z - a, HQ, D), dtype=torch.float64, device="cuda")
    lse = torch.empty((z - a, HQ), dtype=torch.float64, device="cuda")
    for h in range(HKV):
        k, v = (pages[:, x, :, h].reshape(-1, D)[:m].double() for x in (0, 1))
        for u in range(G * h, G * h + G):
            sc = (s.q[a:z, u].double() @ k.T) * SCALE
            sc[hidden] = -math.inf
            lse[:, u] = torch.logsumexp(sc, 1)
            out[:, u] = torch.softmax(sc, 1) @ v
    return out, lse


def exact(case, seed):
    kind = case["kind"]
    if kind == "evict":                                       # rows move, nothing is computed
        return None
    s = prepare(case, seed)
    if kind == "chunk":
        return {"out": torch.cat([_attend64(s, r, case["window"], case["sinks"])[0] for r in range(case["R"])])}
    if kind == "observe":
        scores = s.scores.double()
        for r in range(case["R"]):
            a, z, past = int(s.q_start[r]), int(s.q_start[r + 1]), int(s.kv_start[r])
            m = past + z - a
            pages = s.cache[s.table[r, : -(-m // PAGE)].long()]
            hidden = torch.arange(m, device="cuda")[None] > torch.arange(past, m, device="cuda")[:, None]
            for u in range(HQ):
                k = pages[:, 0, :, u // G].reshape(-1, D)[:m].double()
                sc = (s.q[a:z, u].double() @ k.T) * SCALE - s.lse[a:z, u].double()[:, None]
                sc[hidden] = -math.inf
                scores[r, u // G, :m] += sc.exp().sum(0)
        return {"scores": scores}
    if kind in ("token", "weigh"):
        out = torch.empty((case["B"], HQ, D), dtype=torch.float64, device="cuda")
        lse = torch.empty((case["B"], HQ), dtype=torch.float64, device="cuda")
        scores = s.scores.double() if kind == "weigh" else None
        for b, n in enumerate(s.lens.tolist()):
            j = torch.arange(n, device="cuda")
            if kind == "token":
                j = j[(j >= n - case["window"]) | (j < case["sinks"])]
            kv = s.cache[s.table[b, j // PAGE].long(), :, j % PAGE].double()          # [n, 2, 8, D]
            for h in range(HKV):
                sc = (s.q[b, G * h: G * h + G].double() @ kv[:, 0, h].T) * SCALE
                lse[b, G * h: G * h + G] = torch.logsumexp(sc, 1)
                p = torch.softmax(sc, 1)
                out[b, G * h: G * h + G] = p @ kv[:, 1, h]
                if scores is not None:
                    scores[b, h, :n] += p.sum(0)
        return {"out": out, "lse": lse} if scores is None else {"out": out, "lse": lse, "scores": scores}
    B, S, train = case["B"], case["S"], kind == "train"
    q, k, v = (t.detach().transpose(1, 2) if train else t for t in (s.q, s.k, s.v))
    out = torch.zeros((B, S, HQ, D), dtype=torch.float64, device="cuda")
    dq, dk, dv = (torch.zeros((B, h, S, D), dtype=torch.float64, device="cuda") for h in (HQ, HKV, HKV))
    step = 2048
    for b, n in enumerate(s.lens.tolist()):
        for r in range(0, n, step):
            e = min(n, r + step)
            i = torch.arange(r, e, device="cuda")[:, None]
            j = torch.arange(e, device="cuda")[None]
            hidden = (j > i) | ((j <= i - case["window"]) & (j >= case["sinks"]))
            for u in range(HQ):
                qh, kh, vh = q[b, r:e, u].double(), k[b, :e, u // G].double(), v[b, :e, u // G].double()
                sc = (qh @ kh.T) * SCALE
                sc[hidden] = -math.inf
                p = torch.softmax(sc, 1)
                o = p @ vh
                out[b, r:e, u] = o
                if train:
                    g = s.dout[b, r:e, u].double()
                    dv[b, u // G, :e] += p.T @ g
                    ds = p * (g @ vh.T - (g * o).sum(1, keepdim=True))
                    dq[b, u, r:e] = (ds @ kh) * SCALE
                    dk[b, u // G, :e] += (ds.T @ qh) * SCALE
    return {"out": out, "dq": dq, "dk": dk, "dv": dv} if train else {"out": out}
