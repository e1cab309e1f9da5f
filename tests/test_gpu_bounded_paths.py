"""The paths that call the window, score and eviction kernels: the attention backend of a sliding-window layer, the windowed
baseline of the training wrapper, a HuggingFace model with a sliding window of its own, and the custom ops."""
import copy

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from abridgekv_amd import backend as bk
from abridgekv_amd import ops
from oracle import window as ow

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


def _tables(lens, pool, rng):
    need = [-(-n // 16) for n in lens]
    pages = rng.permutation(pool)[: sum(need)]
    table = np.zeros((len(lens), max(need)), np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = pages[at: at + n]
        at += n
    return table


def _step(seed, qlen, seq, pool=260):
    rng = np.random.default_rng(seed)
    gen = torch.Generator().manual_seed(seed)
    table = _tables(seq, pool, rng)
    cache = torch.randn((pool, 2, 16, 8, 128), generator=gen).to(torch.bfloat16)
    T = sum(qlen)
    q = torch.randn((T, 32 * 128), generator=gen).to(torch.bfloat16)
    k, v = (torch.randn((T, 8 * 128), generator=gen).to(torch.bfloat16) for _ in range(2))
    return table, cache, q, k, v


@pytest.mark.parametrize("window,sinks,max_pages", [(100, 4, 60), (1, 0, 60), (33, 200, 20), (5000, 0, 60)])
def test_backend_step_under_a_window(window, sinks, max_pages):
    qlen, seq = [1, 1, 1, 40, 100], [300, 17, 5, 40, 280]
    table, cache, q, k, v = _step(window, qlen, seq)
    cd = cache.cuda()
    qsl = np.concatenate([[0], np.cumsum(qlen)])
    pos = np.concatenate([np.arange(n - m, n) for n, m in zip(seq, qlen)])
    builder = bk.AbridgeMetadataBuilder(max_num_seqs=8, max_pages=max_pages)
    md = builder.build(qsl, seq, torch.from_numpy(table).cuda(), positions=torch.from_numpy(pos).cuda())
    impl = bk.AbridgeAttentionImpl(sliding_window=window, sinks=sinks)
    lse = torch.empty((sum(qlen), 32), device="cuda")
    out = impl.forward(None, q.cuda(), k.cuda(), v.cuda(), cd, md, output_lse=lse).view(-1, 32, 128)
    now = cd.cpu().double().numpy()
    for r, (m, n) in enumerate(zip(qlen, seq)):
        at = np.arange(n)
        kk, vv = (now[table[r, at // 16], i, at % 16] for i in (0, 1))
        a, z = qsl[r], qsl[r + 1]
        assert (kk[n - m:] == k[a:z].double().numpy().reshape(-1, 8, 128)).all()
        want, want_lse, _, tol = ow.attend(q[a:z].double().numpy().reshape(-1, 32, 128), kk, vv,
                                           ow.visible(np.arange(n - m, n), n, window, sinks), SCALE, True)
        assert (np.abs(out[a:z].double().cpu().numpy() - want) <= tol + 2.0 ** -11 * 5).all(), r
        assert np.abs(lse[a:z].double().cpu().numpy() - want_lse).max() <= ow.SLACK * ow.EPS + 1e-4, r


def test_backend_window_decode_replays_in_a_graph():
    seq = [700, 333, 90, 16]
    table, cache, q, k, v = _step(3, [1] * 4, seq)
    builder = bk.AbridgeMetadataBuilder(max_num_seqs=4, max_pages=table.shape[1])
    md = builder.build(np.arange(5), seq, torch.from_numpy(table).cuda(),
                       positions=torch.tensor([n - 1 for n in seq]).cuda())
    impl = bk.AbridgeAttentionImpl(sliding_window=200, sinks=5)
    base = cache.cuda()
    qs, ks, vs, cg = q.cuda(), k.cuda(), v.cuda(), base.clone()
    out = torch.empty_like(qs)
    impl.forward(None, qs, ks, vs, cg, md, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        impl.forward(None, qs, ks, vs, cg, md, out)
    for i in range(3):
        gen = torch.Generator().manual_seed(i)
        for t in (qs, ks, vs):
            t.copy_(torch.randn(t.shape, generator=gen).to(torch.bfloat16))
        graph.replay()
        ce = base.clone()
        want = impl.forward(None, qs, ks, vs, ce, md)
        torch.cuda.synchronize()
        assert torch.equal(out, want), i


def _model(seed, **kw):
    transformers = pytest.importorskip("transformers")
    torch.manual_seed(seed)
    cfg = transformers.Qwen3Config(vocab_size=257, hidden_size=256, intermediate_size=512, num_hidden_layers=2,
                                   num_attention_heads=32, num_key_value_heads=8, head_dim=128,
                                   max_position_embeddings=4096,
                                   rope_parameters={"rope_theta": 1e6, "rope_type": "default"}, **kw)
    cfg._attn_implementation = "eager"
    return transformers.Qwen3ForCausalLM(cfg).to(torch.bfloat16).eval()


def _dense_windowed(model, ids, window, sinks, dtype):
    """Next-token cross-entropy over all positions but the block ends' of one block, by eager attention with the mask written
    out, and the gradient of the embedding."""
    m = copy.deepcopy(model).to(dtype)
    n = ids.shape[1]
    vis = torch.from_numpy(ow.visible(np.arange(n), n, window, sinks))
    mask = torch.zeros((1, 1, n, n), dtype=dtype).masked_fill(~vis, torch.finfo(dtype).min)
    hid = m.model(inputs_embeds=m.model.embed_tokens(ids), attention_mask={"full_attention": mask}, use_cache=False)
    ce = F.cross_entropy(m.lm_head(hid.last_hidden_state[:, :-1].reshape(-1, 256)).double(), ids[:, 1:].reshape(-1))
    ce.backward()
    return float(ce.detach()), m.model.embed_tokens.weight.grad.double()


def test_windowed_baseline_of_the_training_wrapper():
    """The baseline under a window against eager attention in float64, within twice what the same model in bf16 differs by
    (and 1e-3, as the full-context baseline's test); its gradient likewise."""
    from abridgekv_amd.compress_forward import CompressLM
    base = _model(11)
    ids = torch.randint(0, 257, (2, 1, 192), generator=torch.Generator().manual_seed(1))
    want, grad = _dense_windowed(base, ids[:, 0], 40, 3, torch.float64)
    eager, eager_grad = _dense_windowed(base, ids[:, 0], 40, 3, torch.bfloat16)
    clm = CompressLM(copy.deepcopy(base).cuda(), 192, 1, 16, code_positions="appended")
    got = clm(ids.cuda(), baseline=True, window=40, sinks=3)["ce"]
    assert abs(float(got) - want) <= 2 * abs(eager - want) + 1e-3
    got.backward()
    mine = clm.model.model.embed_tokens.weight.grad.double().cpu()
    assert (mine - grad).norm() <= 2 * (eager_grad - grad).norm() + 1e-3 * grad.norm()
    with torch.no_grad():
        full = clm(ids.cuda(), baseline=True)["ce"]
        wide = clm(ids.cuda(), baseline=True, window=10000)["ce"]
        assert abs(float(full) - float(wide)) <= 2 * abs(eager - want) + 1e-3
        assert abs(float(full) - float(got)) > 0
    with pytest.raises(ValueError, match="window"):
        clm(ids.cuda(), window=40)
    with pytest.raises(ValueError, match="sinks"):
        clm(ids.cuda(), baseline=True, sinks=4)


def test_model_with_its_own_sliding_window():
    """A model whose second layer has a sliding window: its layers' kwarg reaches the kernels."""
    from abridgekv_amd.compress_forward import ATTN_IMPLEMENTATION, register_attention
    base = _model(12, use_sliding_window=True, sliding_window=24, layer_types=["full_attention", "sliding_attention"])
    ids = torch.randint(0, 257, (1, 130), generator=torch.Generator().manual_seed(2))

    def eager(dtype):
        m = copy.deepcopy(base).to(dtype)
        masks = {}
        for name, window in (("full_attention", 130), ("sliding_attention", 24)):
            vis = torch.from_numpy(ow.visible(np.arange(130), 130, window, 0))
            masks[name] = torch.zeros((1, 1, 130, 130), dtype=dtype).masked_fill(~vis, torch.finfo(dtype).min)
        with torch.no_grad():
            return m.model(input_ids=ids, attention_mask=masks, use_cache=False).last_hidden_state.double()

    want, rough = eager(torch.float64), eager(torch.bfloat16)
    register_attention()
    m = copy.deepcopy(base).cuda()
    m.config._attn_implementation = ATTN_IMPLEMENTATION
    with torch.no_grad():
        got = m.model(input_ids=ids.cuda(), attention_mask={"full_attention": None, "sliding_attention": None},
                      use_cache=False).last_hidden_state.double().cpu()
    assert (got - want).norm() <= 2 * (rough - want).norm()


def test_custom_ops_match_direct_calls():
    T = torch.ops.abridgekv
    seq = [300, 17, 90]
    table, cache, q, _, _ = _step(9, [1] * 3, seq)
    q, cache, table = q.view(3, 32, 128).cuda(), cache.cuda(), torch.from_numpy(table).cuda()
    lens = torch.tensor(seq, dtype=torch.int32, device="cuda")
    W = table.shape[1]
    out, lse = torch.empty_like(q), torch.empty((3, 32), device="cuda")
    ws = ops.decode_window_workspace(3, W, 150, 4, 4, device="cuda")
    T.decode_attn_window(q, cache, table, lens, 150, 4, SCALE, W, 4, out, lse, ws)
    want_lse = torch.empty_like(lse)
    want, _ = ops.decode_attention_window(q, cache, table, lens, 150, 4, SCALE, lse=want_lse, split_pages=4)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    with pytest.raises(ValueError, match="workspace"):
        T.decode_attn_window(q, cache, table, lens, 150, 4, SCALE, W, 4, out, lse, None)
    wide = torch.zeros((3, 40), dtype=torch.int32, device="cuda")
    wide[:, :W] = table
    scores = torch.rand((1, 3, 8, 640), device="cuda")
    want_scores = scores.clone()
    T.decode_attn_scored(q, cache, wide, lens, scores[0], SCALE, 40, 8, out, lse,
                         ops.decode_scored_workspace(3, 40, 8, device="cuda"))
    want, _ = ops.decode_attention_scored(q, cache, wide, lens, want_scores[0], SCALE, lse=want_lse, split_pages=8)
    assert torch.equal(out, want) and torch.equal(lse, want_lse) and torch.equal(scores, want_scores)
    with pytest.raises(ValueError, match="workspace"):
        T.decode_attn_scored(q, cache, wide, lens, scores[0], SCALE, 40, 8, out, lse, None)
    positions = torch.full((1, 3, 8, 640), -1, dtype=torch.int32, device="cuda")
    other, want_positions, new = cache.clone(), positions.clone(), torch.empty_like(lens)
    T.kv_evict([cache], wide, lens, scores, positions, lens, 64, 4, 16, 40, new, None)
    want = ops.kv_evict([other], wide, lens, want_scores, want_positions, lens, 64, 4, 16)
    assert torch.equal(new, want) and torch.equal(cache, other)
    assert torch.equal(scores, want_scores) and torch.equal(positions, want_positions)
    gen = torch.Generator().manual_seed(5)
    pq, pk, pv, g = (torch.randn((2, 150, h, 128), generator=gen).to(torch.bfloat16).cuda() for h in (32, 8, 8, 32))
    sl = torch.tensor([150, 61], dtype=torch.int32, device="cuda")
    pout, plse, wlse = torch.empty_like(pq), torch.empty((2, 32, 150), device="cuda"), torch.empty((2, 32, 150), device="cuda")
    T.window_attn(pq, pk, pv, 50, 3, sl, SCALE, pout, plse)
    want, _ = ops.window_attention(pq, pk, pv, 50, 3, seq_lens=sl, scale=SCALE, lse=wlse)
    assert torch.equal(pout, want) and torch.equal(plse, wlse)
    grads = T.window_attn_bwd(pq, pk, pv, pout, plse, g, 50, 3, sl, SCALE)
    assert all(torch.equal(a, b) for a, b in zip(grads, ops.window_attention_backward(pq, pk, pv, want, wlse, g, 50, 3,
                                                                                      seq_lens=sl, scale=SCALE)))
