"""The paths that call the fused norms, the 4-bit cache and the log probabilities: the attention backend, the paged generator, the
training wrapper and the custom ops; and a whole step of them in a row."""
import copy

import numpy as np
import pytest
import torch

from abridgekv_amd import backend as bk
from abridgekv_amd import ops
from oracle import int4 as oi
from oracle import logprobs as olp
from oracle import norm_rope as on
from test_gpu_bounded_paths import _dense_windowed
from test_gpu_gate import _gate, _model

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


def _rows4(cache, table, n):
    """Bytes [n, 2, 640] of a sequence's first n slots."""
    at = np.arange(n)
    return cache.cpu().numpy()[table[at // 16], :, at % 16]


def _visible(n, m, limit=None, excluded=None):
    """[m queries, n rows]: causal, or a code step's key limit without its excluded range."""
    j = np.arange(n)[None]
    if limit is None:
        return j <= np.arange(n - m, n)[:, None]
    vis = np.repeat(j < limit, m, 0)
    if excluded is not None:
        vis[:, excluded[0]: excluded[1]] = False
    return vis


@pytest.mark.parametrize("builder_dtype", ["int4", "auto"])
def test_backend_step_over_4_bits(builder_dtype):
    """Decodes, prompt chunks and a code step with a hidden tail in one batch; the workspace of a 4-bit builder and of a bf16 one."""
    qlen, seq = [1, 1, 1, 40, 100, 64], [900, 17, 1, 40, 280, 364]
    rng = np.random.default_rng(5)
    need = [-(-n // 16) for n in seq]
    pool = sum(need) + 4
    pages = rng.permutation(pool)
    table = np.zeros((len(seq), max(need)), np.int32)
    for b, n in enumerate(need):
        table[b, :n] = pages[sum(need[:b]): sum(need[: b + 1])]
    shape = bk.AbridgeAttentionBackend.get_kv_cache_shape(pool, kv_cache_dtype="int4")
    gen = torch.Generator().manual_seed(6)
    cache = torch.randint(0, 256, shape, dtype=torch.uint8, generator=gen).cuda()
    for b, n in enumerate(seq):                              # what the earlier steps left
        k, v = (torch.randn((n, 8, 128), generator=gen).to(torch.bfloat16).cuda() for _ in range(2))
        at = torch.arange(n)
        slots = torch.from_numpy(table[b].astype(np.int64))[at // 16] * 16 + at % 16
        ops.kv_append_int4(k, v, slots.cuda(), cache)
    T = sum(qlen)
    q, k, v = (torch.randn((T, h * 128), generator=gen).to(torch.bfloat16) for h in (32, 8, 8))
    qsl = np.concatenate([[0], np.cumsum(qlen)])
    pos = np.concatenate([np.arange(n - m, n) for n, m in zip(seq, qlen)])
    builder = bk.AbridgeMetadataBuilder(max_num_seqs=8, max_pages=64, kv_cache_dtype=builder_dtype)
    limits = [bk.NOT_CODE] * 5 + [316]
    ex = [[0, 0]] * 5 + [[280, 300]]
    md = builder.build(qsl, seq, torch.from_numpy(table).cuda(), positions=torch.from_numpy(pos).cuda(), code_key_limit=limits,
                       code_excluded=ex)
    impl = bk.AbridgeAttentionImpl(kv_cache_dtype="int4")
    lse = torch.empty((T, 32), device="cuda")
    out = impl.forward(None, q.cuda(), k.cuda(), v.cuda(), cache, md, output_lse=lse).view(-1, 32, 128)
    for r, (m, n) in enumerate(zip(qlen, seq)):
        rows = _rows4(cache, table[r], n)
        a, z = qsl[r], qsl[r + 1]
        assert np.array_equal(rows[n - m:, 0], oi.quantise(k[a:z].float().numpy().reshape(-1, 8, 128)))
        vis = _visible(n, m, 316 if r == 5 else None, (280, 300))
        want, want_lse, tol, ltol = oi.attend(q[a:z].double().numpy().reshape(-1, 32, 128), rows[:, 0], rows[:, 1], vis, SCALE,
                                              wide=r >= 3)
        assert (np.abs(out[a:z].double().cpu().numpy() - want) <= tol).all(), r
        assert (np.abs(lse[a:z].double().cpu().numpy() - want_lse) <= ltol).all(), r


def test_backend_decode_over_4_bits_replays_in_a_graph():
    seq = [700, 333, 90, 16]
    need = [-(-n // 16) for n in seq]
    table = np.zeros((4, max(need)), np.int32)
    for b, n in enumerate(need):
        table[b, :n] = np.arange(n) + sum(need[:b])
    builder = bk.AbridgeMetadataBuilder(max_num_seqs=4, max_pages=table.shape[1], kv_cache_dtype="int4")
    md = builder.build(np.arange(5), seq, torch.from_numpy(table).cuda(), positions=torch.tensor([n - 1 for n in seq]).cuda())
    impl = bk.AbridgeAttentionImpl(kv_cache_dtype="int4")
    gen = torch.Generator().manual_seed(1)
    base = torch.zeros(ops.kv_cache_int4_shape(sum(need)), dtype=torch.uint8, device="cuda")
    for b, n in enumerate(seq):
        k, v = (torch.randn((n, 8, 128), generator=gen).to(torch.bfloat16).cuda() for _ in range(2))
        ops.kv_append_int4(k, v, torch.arange(n, device="cuda") + 16 * sum(need[:b]), base)
    q, k, v = (torch.randn((4, h * 128), generator=gen).to(torch.bfloat16).cuda() for h in (32, 8, 8))
    out, cg, ce = torch.empty_like(q), base.clone(), base.clone()
    impl.forward(None, q, k, v, cg, md, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        impl.forward(None, q, k, v, cg, md, out)
    for i in range(4):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=gen))
        graph.replay()
        want = impl.forward(None, q, k, v, ce, md)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(cg, ce), i


@pytest.mark.parametrize("T,policy,stepwise", [(0, "static", [1]), (12, "rolling", [0])])
def test_fused_norms_match_dense_forward(T, policy, stepwise):
    """The wrapper and the generator with the norms in the rotation's pass: the gate of the plain ones."""
    _gate(31, 64, 3, 16, "bitrev", [40, 100], [16, 4], stepwise, T, policy, options={"fused_norms": True},
          gen_options={"fused_norms": True})


def test_fused_norms_with_code_projections():
    """Code rows with their own query weights, through the fused attention forward."""
    def move(clm):
        for name, module in clm.named_modules():
            if name.endswith("_proj") and hasattr(module, "code"):
                module.code.weight.add_(torch.randn_like(module.code.weight) * 0.02)

    _gate(32, 64, 3, 16, "appended", [40, 100], [16, 4], [1], options={"fused_norms": True, "code_q_heads": True}, perturb=move,
          gen_options={"fused_norms": True})


def test_training_through_the_fused_operators():
    """Loss and gradient of the full-context baseline with fused norms and cross entropy against eager attention in float64,
    within twice what the same model in bf16 differs by (and 1e-3, as the plain wrapper's test)."""
    from abridgekv_amd.compress_forward import CompressLM
    base = _model(41)
    ids = torch.randint(0, 257, (2, 1, 192), generator=torch.Generator().manual_seed(1))
    want, grad = _dense_windowed(base, ids[:, 0], 192, 0, torch.float64)
    eager, eager_grad = _dense_windowed(base, ids[:, 0], 192, 0, torch.bfloat16)
    clm = CompressLM(copy.deepcopy(base).cuda(), 192, 1, 16, fused_norms=True, fused_ce=True)
    for chunk in (0, 100):
        clm.zero_grad()
        got = clm(ids.cuda(), baseline=True, ce_chunk=chunk)["ce"]
        assert abs(float(got.detach()) - want) <= 2 * abs(eager - want) + 1e-3
        got.backward()
        mine = clm.model.model.embed_tokens.weight.grad.double().cpu()
        assert (mine - grad).norm() <= 2 * (eager_grad - grad).norm() + 1e-3 * grad.norm()
        attn = clm.model.model.layers[0].self_attn
        assert attn.q_norm.weight.grad.abs().sum() > 0 and attn.k_norm.weight.grad.abs().sum() > 0


def test_fused_cross_entropy_is_the_plain_one():
    """Every loss path: the same logits, so the losses differ by fp32 sums alone (1e-5 of ~5.6), the gradients by that and the
    rounding of the logits' gradients to bf16 (2^-8 of each, random: 2^-8 of the norm)."""
    from abridgekv_amd.compress_forward import CompressLM
    base = _model(42)
    ids = torch.randint(0, 257, (2, 3, 64), generator=torch.Generator().manual_seed(1)).cuda()
    mask = torch.ones((2, 3, 64), device="cuda")
    mask[0, 0, :40] = 0
    torch.manual_seed(0)
    plain = CompressLM(copy.deepcopy(base).cuda(), 64, 3, 16, code_positions="bitrev")
    torch.manual_seed(0)
    fast = CompressLM(copy.deepcopy(base).cuda(), 64, 3, 16, code_positions="bitrev", fused_ce=True)
    for kw in ({}, {"ce_chunk": 50}, {"resp_mask": mask}, {"resp_mask": mask, "per_token": True, "include_cross_block": True},
               {"block_ce": True}, {"copy_lambda": 1.0}):
        res, grads = [], []
        for clm in (plain, fast):
            clm.zero_grad()
            out = clm(ids, **kw)
            key = "ce_pt" if "ce_pt" in out else "ce"
            (out[key].mean() + out.get("copy", 0)).backward()
            res.append(out)
            grads.append(clm.model.lm_head.weight.grad.double())
        for name, a in res[0].items():
            assert torch.allclose(a.double(), res[1][name].double(), atol=1e-5, rtol=1e-5), (kw, name)
        assert (grads[0] - grads[1]).norm() <= 2.0 ** -8 * grads[0].norm(), kw


def _generator(base, **kw):
    from abridgekv_amd.compress_forward import CompressLM
    from abridgekv_amd.gen_compress import CompressGen
    torch.manual_seed(3)
    clm = CompressLM(copy.deepcopy(base).cuda(), 64, 3, 16, code_positions="bitrev", head_code_quotas=[[16] * 8, [4] * 8]).eval()
    with torch.no_grad():
        clm.pause.normal_(0, 0.05)
    return CompressGen(clm, torch.device("cuda"), raw_prompt_len=40, head_code_quotas=[[16] * 8, [4] * 8], max_tokens=400, **kw)


def test_generator_in_4_bits(monkeypatch):
    """A generator on a 4-bit cache beside one whose bf16 cache holds the same values (rounded to bf16): the same rows at the same
    places after every compaction (the first layer's are equal, what comes before its attention does not depend on it), and
    logits as close as the formats allow. The bf16 cache's values are off by up to 2^-8 of themselves, which the next layer's rows
    inherit: about 2^-8 |x| / s of their codes (|x| / s < 15: under 6 in 100) come out one step s off. The formats' own
    difference, every value off by up to s / 2, has a mean square of s^2 / 12; that of the codes, 0.06 s^2, is less. So the
    logits are no further apart than those of a bf16 cache without rounding are from them, beside what the gate allows a bf16 path
    (the model's own bf16 error, about 3e-3, twice, and 2e-3)."""
    base = _model(51)
    real, exact = ops.qk_norm_rope_append, False

    def rounded(q, k, v, pos, cs, slots, cache, **kw):
        out = real(q, k, v, pos, cs, slots, cache, **kw)
        if not ops.is_int4_cache(cache) and not exact:
            page, off = slots // 16, slots % 16
            for half in (0, 1):
                rows = oi.values(oi.quantise(cache[page, half, off].float().cpu().numpy()))
                cache[page, half, off] = torch.from_numpy(rows).to(torch.bfloat16).cuda()
        return out

    monkeypatch.setattr(ops, "qk_norm_rope_append", rounded)
    g4, gb, gx = _generator(base, kv_cache_dtype="int4"), _generator(base, fused_norms=True), _generator(base, fused_norms=True)
    ids = torch.randint(0, 257, (3 * 64,), generator=torch.Generator().manual_seed(2)).tolist()
    worst = formats = 0.0
    for blk in range(3):
        toks = ids[64 * blk: 64 * blk + 64]
        h4, hb = (torch.cat([g.feed_content(toks[:60])] + [g.feed_content([t]) for t in toks[60:]]) for g in (g4, gb))
        exact = True
        hx = torch.cat([gx.feed_content(toks[:60])] + [gx.feed_content([t]) for t in toks[60:]])
        gx.compress()
        exact = False
        formats = max(formats, float((gx.lm_head(hx).double() - gb.lm_head(hb).double()).detach().abs().max()))
        l4, lb = (g4.lm_head(h).double() for h in (h4, hb))
        worst = max(worst, float((l4 - lb).detach().abs().max()))
        g4.compress()
        gb.compress()
        assert g4.resident_rows() == gb.resident_rows()
        assert g4.caches[0].shape[-1] == 640
        n = g4.resident_rows()[0]
        table = torch.tensor(g4.planner.get_blocks(g4.rid)[g4.group_of[0]])
        at = torch.arange(n)
        slots = (table[at // 16].long() * 16 + at % 16).cuda()
        k4, v4 = ops.kv_read_int4(g4.caches[g4.tensor_of[0]], slots, torch.bfloat16)
        cb = gb.caches[gb.tensor_of[0]]
        assert torch.equal(k4, cb[slots // 16, 0, slots % 16]) and torch.equal(v4, cb[slots // 16, 1, slots % 16])
    assert worst <= formats + 2 * 3e-3 + 2e-3, (worst, formats)


@pytest.mark.parametrize("kw", [{}, {"kv_cache_dtype": "int4"}])
def test_scores_of_an_answer(kw):
    """score() against the logits of the same chunks, in float64."""
    base = _model(52)
    ids = torch.randint(0, 257, (150,), generator=torch.Generator().manual_seed(4)).tolist()
    got = _generator(base, **kw).score(ids[:50], ids[50:], temperature=0.9, top=3)
    g, logits = _generator(base, **kw), []
    for a, z in ((0, 64), (64, 128), (128, 149)):
        h = g.feed_content(ids[a:z])
        logits.append(g.lm_head(h[max(0, 49 - a):]).double().cpu().detach())
        if g.f == g.C:
            g.compress()
    x, t = torch.cat(logits).numpy(), np.array(ids[50:])
    ls, lp, ent = olp.forward(x, t, 0.9)
    assert got.logprob.shape == (100,) and np.abs(got.logprob.double().cpu().numpy() - lp).max() <= 1e-5
    assert np.abs(got.entropy.double().cpu().numpy() - ent).max() <= 1e-5
    assert np.array_equal(got.top_ids.cpu().numpy(), olp.top(x, 3))
    with pytest.raises(ValueError, match="answer"):
        _generator(base, **kw).score(ids[:5], [])
    one = _generator(base, **kw).score(ids[:1], ids[1:2])
    assert one.logprob.shape == (1,) and one.top_ids.shape == (1, 0)


def test_teacher_forced_scores():
    from abridgekv_amd.compress_forward import CompressLM
    clm = CompressLM(copy.deepcopy(_model(53)).cuda(), 64, 2, 16, code_positions="bitrev").eval()
    ids = torch.randint(0, 257, (2, 2, 64), generator=torch.Generator().manual_seed(1)).cuda()
    x = clm.loss_logits(ids).double().cpu().numpy()
    t = torch.stack([ids[b].reshape(-1)[clm.predict_flat + 1] for b in range(2)]).reshape(-1).cpu().numpy()
    ls, lp, ent = olp.forward(x, t, 1.0)
    for chunk in (4096, 100):
        got = clm.token_logprobs(ids, top=2, chunk=chunk)
        # (a chunk's product may round other logits to bf16: 2^-8 of logits below 2)
        tol = 1e-5 if chunk == 4096 else 2 * 2.0 ** -8 * np.abs(x).max() + 1e-5
        assert np.abs(got.logprob.double().cpu().numpy() - lp).max() <= tol
        assert np.abs(got.entropy.double().cpu().numpy() - ent).max() <= 2 * tol
        if chunk == 4096:
            assert np.array_equal(got.top_ids.cpu().numpy(), olp.top(x, 2))


def test_a_step_of_them_together():
    """Norms, rotation and append into 4 bits, attention, an output product and the log probabilities of the next tokens, twice in a
    row over three sequences, against float64 over the rows that the cache holds."""
    gen = torch.Generator().manual_seed(8)
    lens = [40, 7, 130]
    table = torch.tensor([[3, 9, 1, 0, 0, 0, 0, 0, 0], [5, 0, 0, 0, 0, 0, 0, 0, 0], [2, 4, 6, 8, 10, 12, 14, 0, 7]], dtype=torch.int32)
    cache = torch.zeros(ops.kv_cache_int4_shape(16), dtype=torch.uint8, device="cuda")
    wq, wk = ((1 + 0.2 * torch.randn(128, generator=gen)).to(torch.bfloat16).cuda() for _ in range(2))
    cs = ops.rope_cos_sin_cache(200, device="cuda")
    head = (torch.randn((4096, 1000), generator=gen) / 64).to(torch.bfloat16).cuda()
    n = [0, 0, 0]

    def step(qlen, last):
        T = sum(qlen)
        q, k, v = (torch.randn((T, h, 128), generator=gen).to(torch.bfloat16).cuda() for h in (32, 8, 8))
        pos = torch.cat([torch.arange(a, a + m) for a, m in zip(n, qlen)])
        req = torch.repeat_interleave(torch.arange(3), torch.tensor(qlen))
        slots = (table[req, pos // 16].long() * 16 + pos % 16).cuda()
        qr = ops.qk_norm_rope_append(q, k, v, pos.cuda(), cs, slots, cache, q_weight=wq, k_weight=wk, max_position=199)
        want_q = on.forward(q.double().cpu().numpy(), wq.double().cpu().numpy(), cs[pos.cuda(), None, :64].double().cpu().numpy(),
                            cs[pos.cuda(), None, 64:].double().cpu().numpy(), 1e-6)
        assert np.abs(qr.double().cpu().numpy() - want_q).max() <= 2.0 ** -8 * np.abs(want_q).max() + 1e-5
        for b, m in enumerate(qlen):
            n[b] += m
        if last:
            sl = torch.tensor(n, dtype=torch.int32, device="cuda")
            out, _ = ops.decode_attention_int4(qr, cache, table.cuda(), sl)
        else:
            starts = np.concatenate([[0], np.cumsum(qlen)])
            out, _ = ops.paged_prefill_attention_int4(qr, cache, table.cuda(), starts, [a - m for a, m in zip(n, qlen)], n, True)
        at = 0
        for b, m in enumerate(qlen):
            rows = _rows4(cache, table[b].numpy(), n[b])
            want, _, tol, _ = oi.attend(qr[at: at + m].double().cpu().numpy(), rows[:, 0], rows[:, 1], _visible(n[b], m), SCALE,
                                        wide=not last)
            assert (np.abs(out[at: at + m].double().cpu().numpy() - want) <= tol).all()
            at += m
        logits = out.view(T, -1) @ head
        t = torch.randint(0, 1000, (T,), generator=gen)
        got = ops.token_logprobs(logits, t.cuda(), top=4)
        x = logits.double().cpu().numpy()
        assert np.abs(got.logprob.double().cpu().numpy() - olp.forward(x, t.numpy())[1]).max() <= 1e-5
        assert np.array_equal(got.top_ids.cpu().numpy(), olp.top(x, 4))

    step(lens, False)
    step([1, 1, 1], True)
    step([1, 1, 1], True)


def test_custom_ops_match_direct_calls():
    T = torch.ops.abridgekv
    gen = torch.Generator().manual_seed(5)

    def rand(*shape):
        return torch.randn(shape, generator=gen).to(torch.bfloat16).cuda()

    q, k, v = rand(40, 32, 128), rand(40, 8, 128), rand(40, 8, 128)
    wq, wk = rand(128), rand(128)
    pos = torch.arange(40, device="cuda")
    cs = ops.rope_cos_sin_cache(64, device="cuda")
    a, b = (torch.zeros(ops.kv_cache_int4_shape(4), dtype=torch.uint8, device="cuda") for _ in range(2))
    out = torch.empty_like(q)
    T.qk_norm_rope_append(q, k, v, pos, cs, pos, a, wq, wk, 1e-6, 0, 0, 39, 0, out)
    want = ops.qk_norm_rope_append(q, k, v, pos, cs, pos, b, q_weight=wq, k_weight=wk, max_position=39)
    assert torch.equal(out, want) and torch.equal(a, b)
    T.kv_append_int4(v, k, pos, a)
    ops.kv_append_int4(v, k, pos, b)
    assert torch.equal(a, b)
    table = torch.arange(3, dtype=torch.int32, device="cuda")[None]
    sl = torch.tensor([40], dtype=torch.int32, device="cuda")
    o, lse = torch.empty_like(q[:1]), torch.empty((1, 32), device="cuda")
    with pytest.raises(ValueError, match="workspace"):
        T.decode_attn_int4(q[:1], a, table, sl, SCALE, 3, 2, o, lse, None)
    T.decode_attn_int4(q[:1], a, table, sl, SCALE, 3, 2, o, lse, ops.decode_int4_workspace(1, 3, 2, device="cuda"))
    wlse = torch.empty_like(lse)
    want, _ = ops.decode_attention_int4(q[:1], b, table, sl, SCALE, lse=wlse, split_pages=2)
    assert torch.equal(o, want) and torch.equal(lse, wlse)
    tq, tk, cos = q.view(2, 20, 32, 128), k.view(2, 20, 8, 128), rand(1, 20, 128)
    got, want = T.qk_norm_rope(tq, tk, cos, cos, wq, wk, 1e-6), ops.qk_norm_rope(tq, tk, cos, cos, wq, wk, 1e-6)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    got = T.qk_norm_rope_bwd(tq, tk, tq, tk, cos, cos, wq, wk, 1e-6)
    assert all(torch.equal(x, y) for x, y in zip(got, ops.qk_norm_rope_backward(tq, tk, tq, tk, cos, cos, wq, wk, 1e-6)))
    logits, t = rand(5, 3000), torch.randint(0, 3000, (5,), generator=gen).cuda()
    got, want = T.token_logprobs(logits, t, 0.8, 3), ops.token_logprobs(logits, t, 0.8, top=3, stats=True)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    g = torch.randn(5, device="cuda")
    assert torch.equal(T.token_logprobs_bwd(logits, t, want.stats, g, None, 0.8),
                       ops.token_logprobs_backward(logits, t, want.stats, g, None, 0.8))
