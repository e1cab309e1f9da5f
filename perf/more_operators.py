"""The performance cases of a model's step over a cache held in 4 bits: per-head norms of queries and keys with their
rotation, the 4-bit cache and the attention that reads it, and the log probabilities of the answer.

A case is a dict of plain values; ``kind`` names the call:

  rope    per-head norms and rotation of a serving step's rows, keys and values into the cache
          (``ops.qk_norm_rope_append``)
  train   the same norms and rotation of a training step, with the gradients of q, k and the norms' weights
          (``fused.qk_norm_rope``)
  store   rows written to a 4-bit cache and read back (``ops.kv_append_int4``, ``ops.kv_read_int4``)
  token   one new token per sequence over a 4-bit cache (``ops.decode_attention_int4``)
  chunk   prompt chunks, and code steps behind them, over a 4-bit cache (``ops.paged_prefill_attention_int4``)
  logp    log probabilities of given tokens with entropy and top alternatives (``ops.token_logprobs``)
  loss    the same as a loss, with the gradient of the logits (``fused.token_logprobs``)

Geometry: 32 query heads, 8 KV heads, head size 128, pages of 16 rows. A row of a KV head in 4 bits is 64 bytes of codes
and four pairs (step, minimum) of bf16, one for each 32 dims; a value is minimum + step * code. A slot's row of K (or V) holds
the codes of its 8 heads, then their pairs: 640 bytes. In a head's 16 code words, word 4 * (d // 8 % 4) + d // 32 holds dims
8 * (d // 8) .. + 7, dim d at nibble d % 8 // 2 + 4 * (d % 2). Lengths inside a batch are spread over the case's range in an
order fixed by the case, so that every seed has the same amount of work.
"""
from __future__ import annotations

import math
import types

import numpy as np
import torch

own = False

HQ, HKV, D, PAGE = 32, 8, 128, 16
G = HQ // HKV
ROW4 = HKV * 80                                              # bytes of a slot's K (or V) in 4 bits
SCALE = 1.0 / math.sqrt(D)
EPS = 1e-6


def listed():
    return [
        # one request decoding alone: its token's norms, rotation and append (latency bound)
        {"name": "rope_1", "kind": "rope", "T": 1, "past": 5000, "block_c": 0, "codes_k": 0, "pad": 0},
        # a prompt chunk under the abridged layout, the last rows of the batch padding
        {"name": "rope_2048", "kind": "rope", "T": 2048, "past": 3000, "block_c": 512, "codes_k": 128, "pad": 13},
        # a small training batch of a float32 model, of odd length
        {"name": "train_777", "kind": "train", "dtype": "f32", "B": 3, "S": 777},
        # a training step
        {"name": "train_4096", "kind": "train", "dtype": "bf16", "B": 2, "S": 4096},
        # a decode step of 64 sequences writes its rows (and a reader takes them back)
        {"name": "store_64", "kind": "store", "T": 64},
        # a prompt chunk of odd length
        {"name": "store_1501", "kind": "store", "T": 1501},
        # one request decoding alone over a long context (latency bound)
        {"name": "token_1", "kind": "token", "B": 1, "rows_min": 32000, "rows_max": 32000},
        # a batch of 64 of mixed lengths
        {"name": "token_64", "kind": "token", "B": 64, "rows_min": 500, "rows_max": 9500},
        # a short chunk far into its prompt
        {"name": "chunk_1", "kind": "chunk", "R": 1, "codes": 0, "chunk_min": 61, "chunk_max": 61, "past_min": 4000,
         "past_max": 4000, "quota": 128},
        # a serving step's prompt chunks with a code step of 256 rows behind them
        {"name": "chunk_mix", "kind": "chunk", "R": 4, "codes": 1, "chunk_min": 300, "chunk_max": 512, "past_min": 0,
         "past_max": 8000, "quota": 128},
        # the sampled token of one request with the alternatives that a client asked for
        {"name": "logp_1", "kind": "logp", "dtype": "f32", "T": 1, "V": 131072, "top": 5, "temperature": 0.7},
        # a chunk of a training step's loss
        {"name": "loss_2048", "kind": "loss", "dtype": "bf16", "T": 2048, "V": 131072, "temperature": 1.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "rope", "train", "train", "store", "token", "token", "chunk", "chunk", "logp", "logp", "loss"])
    if kind == "rope":
        T = _log(rng, 1, 2048)
        c = rng.choice([0, 0, 64, 512])
        return {"kind": kind, "T": T, "past": rng.choice([0, _log(rng, 1, 30000)]), "block_c": c, "codes_k": c // 4,
                "pad": rng.choice([0, rng.randint(0, min(T, 20))])}
    if kind == "train":
        f32 = rng.random() < 0.3
        S = _log(rng, 1, 2000 if f32 else 4096)
        return {"kind": kind, "dtype": "f32" if f32 else "bf16", "S": S,
                "B": rng.randint(1, max(1, min(8, (4096 if f32 else 8192) // S)))}
    if kind == "store":
        return {"kind": kind, "T": _log(rng, 1, 2048)}
    if kind == "token":
        B = _log(rng, 1, 64)
        most = min(32000, 500000 // B)
        lo, hi = sorted((_log(rng, 1, most), _log(rng, 1, most)))
        return {"kind": kind, "B": B, "rows_min": lo, "rows_max": hi}
    if kind == "chunk":
        lo, hi = sorted((_log(rng, 1, 512), _log(rng, 2, 512)))
        R = rng.randint(1, 4)
        return {"kind": kind, "R": R, "codes": rng.randint(0, min(2, R)), "chunk_min": lo, "chunk_max": hi, "past_min": 0,
                "past_max": rng.choice([0, _log(rng, 1, 8000)]), "quota": rng.choice([64, 128, 256])}
    V = _log(rng, 250, 131072)
    f32 = rng.random() < 0.5
    T = _log(rng, 1, min(4096, (1 << (27 if kind == "logp" or f32 else 28)) // V))
    case = {"kind": kind, "dtype": "f32" if f32 else "bf16", "T": T, "V": V, "temperature": rng.choice([1.0, 1.0, 0.6, 1.3])}
    if kind == "logp":
        case["top"] = rng.choice([0, 1, 5, 20])
    return case


# -- sizes and inputs ------------------------------------------------------------------------------------------------
def _spread(n, lo, hi, salt):
    """n lengths over [lo, hi], both ends among them (n > 1), in an order fixed by the sizes."""
    v = np.round(np.linspace(lo, hi, n)).astype(np.int64) if n > 1 else np.array([hi], np.int64)
    return np.random.RandomState(17 * n + salt).permutation(v)


def _chunks(case):
    """Queries of each request, the rows before them, the keys each request sees at most, and which are causal: the last
    ``codes`` are code steps of 256 rows, whose queries see the rows before them and ``quota`` of their own."""
    n = _spread(case["R"], case["chunk_min"], case["chunk_max"], 3)
    past = _spread(case["R"], case["past_min"], case["past_max"], 4)
    causal = np.arange(case["R"]) < case["R"] - case["codes"]
    n = np.where(causal, n, 256)
    return n, past, np.where(causal, past + n, past + case["quota"]), causal


def _dtype(case):
    return torch.float32 if case.get("dtype") == "f32" else torch.bfloat16


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


def _angles(n, first=0):
    """cos | sin [n, 128] float32 of the positions from ``first`` on."""
    freq = 1e6 ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
    a = (first + torch.arange(n, dtype=torch.float64, device="cuda"))[:, None] * freq
    return torch.cat([a.cos(), a.sin()], 1).float()


def _rows(gen, n, loud):
    """K or V rows [n, 8, 128] bf16; keys have a few dims that are loud in every row."""
    x = _randn(gen, (n, HKV, D), torch.float32)
    return (x + loud if loud is not None else x).to(torch.bfloat16)


def _loud(gen):
    x = torch.zeros((HKV, D), device="cuda")
    return x.scatter_(1, torch.randint(0, D, (HKV, 4), generator=gen, device="cuda"), 6.0)


def prepare(case, seed):
    s = types.SimpleNamespace(case=case)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 1000003 + 11)
    kind, dt = case["kind"], _dtype(case)
    if kind in ("rope", "store"):
        T = case["T"]
        table, pool = _paged(gen, [T])
        t = torch.arange(T, device="cuda")
        s.slots = table[0, t // PAGE].long() * PAGE + t % PAGE
        s.v = _rows(gen, T, None)
        if kind == "store":
            s.k = _rows(gen, T, _loud(gen))
            s.cache = torch.zeros((pool, 2, PAGE, ROW4), dtype=torch.uint8, device="cuda")
            return s
        if case["pad"]:
            s.slots[T - case["pad"]:] = -1
        s.q, s.k = _randn(gen, (T, HQ, D)), _randn(gen, (T, HKV, D))
        s.wq, s.wk = (1 + 0.2 * _randn(gen, (D,), torch.float32)).to(dt), (1 + 0.2 * _randn(gen, (D,), torch.float32)).to(dt)
        s.positions = case["past"] + t
        s.cos_sin = _angles(case["past"] + T)
        s.cache = torch.zeros((pool, 2, PAGE, HKV, D), dtype=torch.bfloat16, device="cuda")
        return s
    if kind == "train":
        B, S = case["B"], case["S"]
        s.q, s.k, s.dq, s.dk = (_randn(gen, (B, S, h, D), dt) for h in (HQ, HKV, HQ, HKV))
        s.wq, s.wk = ((1 + 0.2 * _randn(gen, (D,), torch.float32)).to(dt) for _ in range(2))
        for x in (s.q, s.k, s.wq, s.wk):
            x.requires_grad_(True)
        cs = _angles(S)
        s.cos, s.sin = (torch.cat([x, x], 1)[None].to(dt) for x in (cs[:, :64], cs[:, 64:]))    # as a model hands them
        return s
    if kind in ("token", "chunk"):
        if kind == "token":
            lens = _spread(case["B"], case["rows_min"], case["rows_max"], 2)
            s.lens = torch.from_numpy(lens.astype(np.int32)).cuda()
            nq = case["B"]
        else:
            n, past, s.kv_limit, s.causal = _chunks(case)
            s.q_start, s.kv_start = np.concatenate([[0], np.cumsum(n)]), past
            lens, nq = past + n, int(n.sum())
        s.table, pool = _paged(gen, lens)
        s.cache = torch.randint(0, 256, (pool, 2, PAGE, ROW4), generator=gen, device="cuda", dtype=torch.uint8)
        loud = _loud(gen)
        used = torch.cat([s.table[b, : -(-int(x) // PAGE)] for b, x in enumerate(lens)]).long()
        for a in range(0, len(used), 2048):                  # pages no sequence holds keep arbitrary bytes
            p = used[a: a + 2048]
            for half, shift in ((0, loud), (1, None)):
                s.cache[p, half] = _pack4(_rows(gen, len(p) * PAGE, shift)).view(len(p), PAGE, ROW4)
        s.q = _randn(gen, (nq, HQ, D))
        return s
    T, V = case["T"], case["V"]
    s.logits = _randn(gen, (T, V), torch.float32).mul_(2.5).to(dt)
    banned = torch.randint(0, V, (V // 500,), generator=gen, device="cuda")     # tokens that may not be sampled
    s.logits[:, banned] = -math.inf
    s.targets = torch.randint(0, V, (T,), generator=gen, device="cuda")
    s.targets = torch.where(torch.isin(s.targets, banned), torch.argmax(s.logits, 1), s.targets)
    if kind == "loss":
        if T > 8:
            s.targets[:: 8] = -100                           # rows without a target
        s.logits.requires_grad_(True)
        s.dlogp = torch.full((T,), -1.0 / T, device="cuda")
        s.dent = torch.full((T,), 0.01 / T, device="cuda")
    return s


# -- one pass --------------------------------------------------------------------------------------------------------
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from abridgekv_amd import fused, ops

    case = s.case
    kind = case["kind"]
    if kind == "rope":
        q = ops.qk_norm_rope_append(s.q, s.k, s.v, s.positions, s.cos_sin, s.slots, s.cache, q_weight=s.wq, k_weight=s.wk,
                                    eps=EPS, block_c=case["block_c"], codes_k=case["codes_k"],
                                    max_position=case["past"] + case["T"] - 1)
        return {"q": q, "cache": s.cache}
    if kind == "train":
        q, k = fused.qk_norm_rope(s.q, s.k, s.cos, s.sin, s.wq, s.wk, EPS)
        grads = torch.autograd.grad((q, k), (s.q, s.k, s.wq, s.wk), (s.dq, s.dk))
        return dict(zip(("q", "k", "dq", "dk", "dwq", "dwk"), (q, k, *grads)))
    if kind == "store":
        ops.kv_append_int4(s.k, s.v, s.slots, s.cache)
        k, v = ops.kv_read_int4(s.cache, s.slots)
        return {"k": k, "v": v}
    if kind == "token":
        lse = torch.empty((case["B"], HQ), device="cuda")
        out, _ = ops.decode_attention_int4(s.q, s.cache, s.table, s.lens, SCALE, lse=lse)
        return {"out": out, "lse": lse}
    if kind == "chunk":
        return {"out": ops.paged_prefill_attention_int4(s.q, s.cache, s.table, s.q_start, s.kv_start, s.kv_limit, s.causal,
                                                        SCALE)[0]}
    if kind == "logp":
        got = ops.token_logprobs(s.logits, s.targets, temperature=case["temperature"], top=case["top"])
        return {"logprob": got.logprob, "entropy": got.entropy, "top_ids": got.top_ids, "top_logprobs": got.top_logprobs}
    logp, ent = fused.token_logprobs(s.logits, s.targets, temperature=case["temperature"])
    (grad,) = torch.autograd.grad((logp, ent), (s.logits,), (s.dlogp, s.dent))
    return {"logprob": logp, "entropy": ent, "dlogits": grad}


def _nibbles():
    """Byte of a head's 64 and shift inside it for each dim."""
    d = torch.arange(D, device="cuda")
    nib = d % 8 // 2 + 4 * (d % 2)
    return 4 * (4 * (d // 8 % 4) + d // 32) + nib // 2, (4 * (nib % 2)).to(torch.uint8)


def _codes4(x):
    """Steps, minima and codes of rows x [n, 8, 128], in float32."""
    g = x.float().view(-1, HKV, 4, 32)
    lo, hi = g.amin(-1), g.amax(-1)
    step = ((hi - lo) / torch.full_like(hi, 15.0)).to(torch.bfloat16).float()      # (by a tensor: an IEEE quotient)
    code = torch.where(step[..., None] > 0, torch.round((g - lo[..., None]) / step[..., None]).clamp(0, 15), 0.0)
    return step, lo, code


def _pack4(x):
    """Rows [n, 8, 128] as [n, 640] bytes."""
    step, lo, code = _codes4(x)
    byte, shift = _nibbles()
    bits = code.view(-1, HKV, D).to(torch.uint8) << shift
    codes = torch.zeros((len(bits), HKV, 64), dtype=torch.uint8, device="cuda")
    even = shift == 0
    codes[..., byte[even]] = bits[..., even]
    codes[..., byte[~even]] += bits[..., ~even]
    pairs = torch.stack([step, lo], -1).to(torch.bfloat16).contiguous().view(torch.uint8)
    return torch.cat([codes.view(-1, 512), pairs.view(-1, 128)], 1)


def _unpack4(rows):
    """[..., 640] bytes as float32 [..., 8, 128]."""
    lead = rows.shape[:-1]
    byte, shift = _nibbles()
    codes = rows[..., :512].view(*lead, HKV, 64)
    vals = ((codes[..., byte] >> shift) & 15).float().view(*lead, HKV, 4, 32)
    pairs = rows[..., 512:].contiguous().view(torch.bfloat16).view(*lead, HKV, 4, 2).float()
    return (pairs[..., 1:] + pairs[..., :1] * vals).view(*lead, HKV, D)


def _softmax(sc, vis):
    """Weights and lse of scores sc [..., keys] where vis holds; rows that see nothing have weights 0 and lse -inf."""
    sc = sc.masked_fill_(~vis, -math.inf)
    m = sc.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = sc.sub_(m).exp_()
    z = p.sum(-1, keepdim=True)
    return p.div_(torch.where(z == 0, 1.0, z)), (torch.log(z) + m)[..., 0]


def _cached(cache, table, n):
    """K and V [B, 8, n, D] float32 of the first n slots of each sequence."""
    j = torch.arange(n, device="cuda")
    kv = _unpack4(cache[table[:, j // PAGE].long(), :, j % PAGE])                   # [B, n, 2, 8, D]
    return kv[:, :, 0].transpose(1, 2).contiguous(), kv[:, :, 1].transpose(1, 2).contiguous()


def _rotated(x, c, sn):
    """Rows x [..., 128] rotated by angles c, sn [..., 64]."""
    a, b = x[..., :64], x[..., 64:]
    return torch.cat([a * c - b * sn, b * c + a * sn], -1)


def _code_positions(positions, block_c, codes_k):
    """RoPE positions of the abridged layout's logical positions: a block's code rows spread over its content rows by
    bit-reversed offsets."""
    if not block_c:
        return positions
    blk, w = positions // (block_c + codes_k), positions % (block_c + codes_k)
    k, rev = (w - block_c).clamp(min=0), torch.zeros_like(w)
    for i in range(codes_k.bit_length() - 1):
        rev = rev * 2 + (k >> i) % 2
    return blk * block_c + torch.where(w < block_c, w, rev * block_c // codes_k)


def _run_plain(s):
    case = s.case
    kind = case["kind"]
    if kind == "rope":
        cs = s.cos_sin[_code_positions(s.positions, case["block_c"], case["codes_k"])][:, None]
        out = []
        for x, w in ((s.q.float(), s.wq), (s.k.float(), s.wk)):
            r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
            out.append(_rotated(x * r * w.float(), cs[..., :64], cs[..., 64:]).to(torch.bfloat16))
        real = s.slots >= 0
        at = s.slots[real]
        s.cache[at // PAGE, :, at % PAGE] = torch.stack([out[1][real], s.v[real]], 1)
        return {"q": out[0], "cache": s.cache}
    if kind == "train":
        c, sn = s.cos.float()[:, :, None, :64], s.sin.float()[:, :, None, :64]
        got = []
        for leaf, weight, dout in ((s.q, s.wq, s.dq), (s.k, s.wk, s.dk)):
            x, w = leaf.detach().float(), weight.detach().float()
            r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
            xh = x * r
            dy = _rotated(dout.float(), c, -sn)
            g = dy * w
            dx = r * (g - xh * (g * xh).mean(-1, keepdim=True))
            dw = (dy * xh).sum((0, 1, 2), dtype=torch.float64)
            got.append([t.to(leaf.dtype) for t in (_rotated(xh * w, c, sn), dx, dw)])
        return {"q": got[0][0], "k": got[1][0], "dq": got[0][1], "dk": got[1][1], "dwq": got[0][2], "dwk": got[1][2]}
    if kind == "store":
        out = []
        for half, x in ((0, s.k), (1, s.v)):
            s.cache[s.slots // PAGE, half, s.slots % PAGE] = _pack4(x)
            out.append(_unpack4(s.cache[s.slots // PAGE, half, s.slots % PAGE]))
        return {"k": out[0], "v": out[1]}
    if kind == "token":
        n = int(case["rows_max"])
        k, v = _cached(s.cache, s.table, n)
        vis = torch.arange(n, device="cuda")[None] < s.lens[:, None]
        p, lse = _softmax(torch.matmul(s.q.float().view(-1, HKV, G, D), k.transpose(2, 3).contiguous()).mul_(SCALE),
                          vis[:, None, None])
        # a page's rows behind its sequence's last hold what an earlier owner left
        v = torch.where(vis[:, None, :, None], v, 0.0)
        return {"out": torch.matmul(p, v).reshape(-1, HQ, D).to(torch.bfloat16), "lse": lse.reshape(-1, HQ)}
    if kind == "chunk":
        out = torch.empty_like(s.q)
        for r in range(case["R"]):
            a, z, past, m = (int(x) for x in (s.q_start[r], s.q_start[r + 1], s.kv_start[r], s.kv_limit[r]))
            k, v = _cached(s.cache, s.table[r: r + 1], m)
            q = s.q[a:z].float().view(1, z - a, HKV, G, D).permute(0, 2, 3, 1, 4).reshape(1, HKV, G * (z - a), D)
            j = torch.arange(m, device="cuda")[None]
            vis = (j <= torch.arange(past, past + z - a, device="cuda")[:, None]) | (not s.causal[r])
            p, _ = _softmax(torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(SCALE), vis.repeat(G, 1))
            o = torch.matmul(p, v).view(HKV, G, z - a, D).permute(2, 0, 1, 3).reshape(z - a, HQ, D)
            out[a:z] = o.to(torch.bfloat16)
        return {"out": out}
    x = s.logits.detach().float() / case["temperature"]
    m = x.amax(1, keepdim=True)
    e = (x - m).exp_()
    z = e.sum(1, keepdim=True)
    lse = z.log() + m
    real = s.targets >= 0
    at = s.targets.clamp(min=0)[:, None]
    logp = torch.where(real, (x.gather(1, at) - lse)[:, 0], 0.0)
    p = e.div_(z)
    ent = lse[:, 0] - torch.where(p > 0, p * x, 0.0).sum(1)
    if kind == "logp":
        ids = torch.sort(s.logits, dim=1, descending=True, stable=True)[1][:, : case["top"]].contiguous()
        return {"logprob": logp, "entropy": ent, "top_ids": ids, "top_logprobs": x.gather(1, ids) - lse}
    g = torch.where(real, s.dlogp, 0.0)[:, None]
    d = p * torch.where(p > 0, -g - s.dent[:, None] * (x - lse + ent[:, None]), 0.0)
    d.scatter_add_(1, at, g)
    return {"logprob": logp, "entropy": ent, "dlogits": (d / case["temperature"]).to(s.logits.dtype)}


# -- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    e = 4 if case.get("dtype") == "f32" else 2
    if kind == "rope":                                       # q, k, v and the angles in, q and a cached row out
        T = case["T"]
        return {"bytes": T * (HQ + 2 * HKV) * D * 2 * 2 + T * (4 * D + 16), "flops": T * (HQ + HKV) * D * 7}
    if kind == "train":                                      # forward in and out; backward rows and gradients in, gradients out
        rows = case["B"] * case["S"] * (HQ + HKV)
        return {"bytes": rows * D * e * 5 + case["S"] * D * 4 * e, "flops": rows * D * 24}
    if kind == "store":                                      # bf16 in, 4 bits out and in, float32 out
        return {"bytes": case["T"] * (2 * HKV * D * 6 + 4 * ROW4), "flops": case["T"] * 2 * HKV * D * 6}
    if kind == "token":
        n = int(_spread(case["B"], case["rows_min"], case["rows_max"], 2).sum())
        return {"bytes": n * 2 * ROW4 + case["B"] * HQ * (2 * D * 2 + 4), "flops": 4 * D * HQ * n}
    if kind == "chunk":
        n, past, limit, causal = _chunks(case)
        pairs = np.where(causal, n * past + n * (n + 1) // 2, n * limit)
        return {"bytes": int(limit.sum()) * 2 * ROW4 + int(n.sum()) * HQ * D * 4, "flops": 4 * D * HQ * int(pairs.sum())}
    size = case["T"] * case["V"]
    if kind == "logp":
        return {"bytes": size * e + case["T"] * (16 + 12 * case["top"]), "flops": 5 * size}
    return {"bytes": 3 * size * e + case["T"] * 32, "flops": 12 * size}


# -- the same results in 64 bits -------------------------------------------------------------------------------------
def _values64(rows):
    """[n, 640] bytes as float64 [n, 8, 128], word by word."""
    words = rows[:, :512].contiguous().view(torch.int32).long().view(-1, HKV, 16) & 0xFFFFFFFF
    pairs = rows[:, 512:].contiguous().view(torch.bfloat16).double().view(-1, HKV, 4, 2)
    out = torch.empty((len(rows), HKV, D), dtype=torch.float64, device="cuda")
    for word in range(16):
        group = word % 4
        for i in range(8):
            code = (words[..., word] >> (4 * (i // 2) + 16 * (i % 2))) & 15
            out[..., 32 * group + 8 * (word // 4) + i] = pairs[..., group, 1] + pairs[..., group, 0] * code
    return out


def _attend64(s, r, q, n, first=None):
    """Out [m, 32, D] and lse [m, 32] float64 of queries q over the first n rows of sequence r; causal from row ``first`` on."""
    pages = s.cache[s.table[r, : -(-n // PAGE)].long()]
    k, v = (_values64(pages[:, x].reshape(-1, ROW4)[:n]) for x in (0, 1))
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(q.shape[:2], dtype=torch.float64, device="cuda")
    for u in range(HQ):
        sc = (q[:, u].double() @ k[:, u // G].T) * SCALE
        if first is not None:
            sc[torch.arange(n, device="cuda")[None] > torch.arange(first, first + len(q), device="cuda")[:, None]] = -math.inf
        lse[:, u] = torch.logsumexp(sc, 1)
        out[:, u] = torch.softmax(sc, 1) @ v[:, u // G]
    return out, lse


def exact(case, seed):
    kind = case["kind"]
    s = prepare(case, seed)
    if kind in ("rope", "train"):
        def rotate(y, angle_c, angle_s):
            z = torch.complex(y[..., :64], y[..., 64:]) * torch.complex(angle_c, angle_s)
            return torch.cat([z.real, z.imag], -1)

        def forward(x, w, angle_c, angle_s):
            return rotate(x / (x.square().sum(-1, keepdim=True) / D + EPS).sqrt() * w, angle_c, angle_s)

        if kind == "rope":
            pos = s.positions.tolist()
            if case["block_c"]:
                c, k = case["block_c"], case["codes_k"]
                bits = k.bit_length() - 1
                for t, p in enumerate(pos):
                    blk, w = divmod(p, c + k)
                    pos[t] = blk * c + (w if w < c else int(f"{w - c:0{bits}b}"[::-1], 2) * c // k)
            cs = s.cos_sin[torch.tensor(pos, device="cuda")].double()[:, None]
            q, k = (forward(x.double(), w.double(), cs[..., :64], cs[..., 64:]) for x, w in ((s.q, s.wq), (s.k, s.wk)))
            cache = s.cache.double()
            real = s.slots >= 0
            flat = cache.view(-1, 2, PAGE, HKV, D)
            flat[s.slots[real] // PAGE, 0, s.slots[real] % PAGE] = k[real]
            flat[s.slots[real] // PAGE, 1, s.slots[real] % PAGE] = s.v[real].double()
            return {"q": q, "cache": cache}
        c, sn = s.cos.double()[:, :, None, :64], s.sin.double()[:, :, None, :64]
        res = {}
        for name, x, w, dout in (("q", s.q, s.wq, s.dq), ("k", s.k, s.wk, s.dk)):
            x, w = x.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
            y = forward(x, w, c, sn)
            dx, dw = torch.autograd.grad(y, (x, w), dout.double())
            res.update({name: y.detach(), "d" + name: dx, "dw" + name: dw})
        return {name: res[name] for name in ("q", "k", "dq", "dk", "dwq", "dwk")}
    if kind == "store":
        out = {}
        for name, x in (("k", s.k), ("v", s.v)):
            g = x.double().view(-1, HKV, 4, 32)
            lo, hi = g.min(-1, keepdim=True)[0], g.max(-1, keepdim=True)[0]
            step = ((hi - lo).float() / torch.full_like(hi, 15.0).float()).to(torch.bfloat16).double()
            code = torch.round((g - lo) / step.clamp(min=1e-300)).clamp(0, 15)
            out[name] = (lo + step * code).view(-1, HKV, D)
        return out
    if kind == "token":
        got = [_attend64(s, b, s.q[b: b + 1], n) for b, n in enumerate(s.lens.tolist())]
        return {"out": torch.cat([o for o, _ in got]), "lse": torch.cat([x for _, x in got])}
    if kind == "chunk":
        got = [_attend64(s, r, s.q[s.q_start[r]: s.q_start[r + 1]], int(s.kv_limit[r]),
                         int(s.kv_start[r]) if s.causal[r] else None)[0] for r in range(case["R"])]
        return {"out": torch.cat(got)}
    T, real = case["T"], s.targets >= 0
    logits = s.logits.detach()
    res = {"logprob": torch.zeros(T, dtype=torch.float64, device="cuda"), "entropy": torch.empty(T, dtype=torch.float64, device="cuda")}
    if kind == "logp":
        res["top_ids"] = torch.empty((T, case["top"]), dtype=torch.int64, device="cuda")
        res["top_logprobs"] = torch.empty((T, case["top"]), dtype=torch.float64, device="cuda")
    else:
        res["dlogits"] = torch.empty(logits.shape, dtype=torch.float64, device="cuda")
    for a in range(0, T, 256):
        z = min(T, a + 256)
        ls = torch.log_softmax(logits[a:z].double() / case["temperature"], 1)
        p = ls.exp()
        ent = -torch.where(p > 0, p * ls, 0.0).sum(1)
        res["entropy"][a:z] = ent
        rows, at = torch.arange(z - a, device="cuda")[real[a:z]], s.targets[a:z][real[a:z]]
        res["logprob"][a:z][rows] = ls[rows, at]
        if kind == "logp":
            ids = torch.sort(ls, dim=1, descending=True, stable=True)[1][:, : case["top"]]
            res["top_ids"][a:z], res["top_logprobs"][a:z] = ids, ls.gather(1, ids)
            continue
        g = torch.where(real[a:z], s.dlogp[a:z].double(), 0.0)[:, None]
        d = torch.where(p > 0, -p * (g + s.dent[a:z].double()[:, None] * (ls + ent[:, None])), 0.0)
        d[rows, at] += g[rows, 0]
        res["dlogits"][a:z] = d / case["temperature"]
    return res
