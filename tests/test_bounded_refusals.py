"""What the window, score and eviction entry points refuse, on the CPU: every bad argument is named before any launch, and
good ones get as far as the device check. The C entry points return an error code for theirs."""
import ctypes as C

import numpy as np
import pytest
import torch

from abridgekv_amd import backend as bk
from abridgekv_amd import ops
from abridgekv_amd._lib import lib

BF, F32, I32 = torch.bfloat16, torch.float32, torch.int32


def _dense(B=2, S=9, dt=BF):
    return [torch.zeros((B, S, h, 128), dtype=dt) for h in (32, 8, 8)]


def _bad(match, call, *a, **k):
    with pytest.raises(ValueError, match=match):
        call(*a, **k)


def test_window_attention():
    q, k, v = _dense()
    on_gpu = "current GPU"
    _bad(on_gpu, ops.window_attention, q, k, v, 4)
    _bad(on_gpu, ops.window_attention, q.float(), k.float(), v.float(), 4, 2, lse=torch.zeros(2, 32, 9))
    for window, sinks in ((0, 0), (-1, 0), (1 << 31, 0), (4, -1), (4, 1 << 31), (2.5, 0), (4, 0.5)):
        _bad("window", ops.window_attention, q, k, v, window, sinks)
    _bad("q must be", ops.window_attention, q[0], k, v, 4)
    _bad("k must be", ops.window_attention, q, k[:, :8], v, 4)
    _bad("v must be", ops.window_attention, q, k, v.float(), 4)
    _bad("q must be", ops.window_attention, q.half(), k, v, 4)
    _bad("k must be", ops.window_attention, q, torch.zeros(2, 9, 4, 128, dtype=BF), v, 4)
    wide = torch.zeros((2, 9, 32, 132), dtype=BF)                         # rows that are not 16-byte aligned
    _bad("aligned", ops.window_attention, wide[..., :128], k, v, 4)
    _bad("aligned", ops.window_attention, torch.zeros((2, 9, 32, 136), dtype=BF)[..., 1:129], k, v, 4)
    _bad("aligned", ops.window_attention, torch.zeros((2, 9, 128, 32), dtype=BF).transpose(2, 3), k, v, 4)
    _bad("seq_lens", ops.window_attention, q, k, v, 4, seq_lens=torch.zeros(3, dtype=I32))
    _bad("seq_lens", ops.window_attention, q, k, v, 4, seq_lens=torch.zeros(2, dtype=torch.int64))
    _bad("seq_lens", ops.window_attention, q, k, v, 4, seq_lens=torch.zeros(4, dtype=I32)[::2])
    _bad("out must be", ops.window_attention, q, k, v, 4, out=torch.zeros_like(q, dtype=F32))
    _bad("lse", ops.window_attention, q, k, v, 4, lse=torch.zeros(2, 9, 32))
    _bad("lse", ops.window_attention_backward, q, k, v, q, torch.zeros(2, 9, 32), q, 4)
    _bad("dout", ops.window_attention_backward, q, k, v, q, torch.zeros(2, 32, 9), q[:, :, :8], 4)
    _bad("out must be", ops.window_attention_backward, q, k, v, q.float(), torch.zeros(2, 32, 9), q, 4)
    _bad(on_gpu, ops.window_attention_backward, q, k, v, q, torch.zeros(2, 32, 9), q, 4)
    low = torch.zeros((2, 9, 32, 128), dtype=torch.float8_e5m2)
    _bad(on_gpu, ops.window_attention, q, k, v, 4, out_low=low)
    for bad in (low[:1], low.view(torch.uint8), low.transpose(1, 2)):
        _bad("out_low", ops.window_attention, q, k, v, 4, out_low=bad)
        _bad("out_low", ops.window_attention_backward, q, k, v, q, torch.zeros(2, 32, 9), q, 4, out_low=bad)
    _bad("out_low", ops.window_attention, q.float(), k.float(), v.float(), 4, out_low=low)


@pytest.mark.parametrize("scale", [0.0, -0.1, float("inf"), float("nan")])
def test_scales(scale):
    """Scores are masked before they are scaled."""
    q, k, v = _dense()
    lse = torch.zeros(2, 32, 9)
    _bad("scale", ops.window_attention, q, k, v, 4, scale=scale)
    _bad("scale", ops.window_attention_backward, q, k, v, q, lse, q, 4, scale=scale)
    q, cache, table, lens = _paged()
    _bad("scale", ops.decode_attention_window, q, cache, table, lens, 4, scale=scale)
    _bad("scale", ops.decode_attention_scored, q, cache, table, lens, torch.zeros((2, 8, 64)), scale=scale)
    _bad("scale", ops.paged_prefill_attention_window, q, cache, table, [0, 2], [0], 4, scale=scale)
    _bad("scale", ops.paged_prefill_scores, q, cache, table, [0, 2], [0], torch.zeros(2, 32), torch.zeros((1, 8, 64)), scale=scale)


def test_outputs_that_share_memory():
    q, k, v = _dense()
    for out in (q[:1].expand(2, -1, -1, -1), q[:, :1].expand(-1, 9, -1, -1), q[:, :, :1].expand(-1, -1, 32, -1),
                torch.zeros(1 << 18, dtype=BF).as_strided((2, 9, 32, 128), (9 * 4096 - 128, 4096, 128, 1))):
        _bad("out must not share", ops.window_attention, q, k, v, 4, out=out)
    order = torch.zeros((32, 9, 2, 128), dtype=BF).permute(2, 1, 0, 3)                 # any order of its own rows
    _bad("current GPU", ops.window_attention, q, k, v, 4, out=order)
    q, cache, table, lens = _paged()
    _bad("out must not share", ops.decode_attention_window, q, cache, table, lens, 4, out=q[:1].expand(2, -1, -1))
    _bad("out must not share", ops.paged_prefill_attention_window, q, cache, table, [0, 2], [0], 4, out=q[:1].expand(2, -1, -1))
    scores, positions = torch.zeros((1, 2, 8, 64)), torch.zeros((1, 2, 8, 64), dtype=I32)
    many = torch.zeros(5, dtype=I32)
    for tokens, out in ((lens.clone(), lens), (many[:2], many[1:3]), (many[1:3], many[:2]), (many[:2], many[:2])):
        _bad("out must be contiguous int32", ops.kv_evict, [cache], table, lens, scores, positions, tokens, 4, out=out)
    _bad("current GPU", ops.kv_evict, [cache], table, lens, scores, positions, many[:2], 4, out=many[2:4])
    _bad("share memory", ops.kv_evict, [cache], table, lens, scores, scores.view(I32), lens.clone(), 4)
    pool = torch.zeros((15, 2, 16, 8, 128), dtype=BF)
    two = dict(scores=torch.zeros((2, 2, 8, 64)), positions=torch.zeros((2, 2, 8, 64), dtype=I32))
    _bad("current GPU", ops.kv_evict, [pool[5:10], pool[:5]], table, lens, num_tokens=lens.clone(), budget=4, **two)


def _paged(B=2, W=4, P=10):
    return (torch.zeros((B, 32, 128), dtype=BF), torch.zeros((P, 2, 16, 8, 128), dtype=BF), torch.zeros((B, W), dtype=I32),
            torch.ones(B, dtype=I32))


@pytest.mark.parametrize("scored", [False, True])
def test_decode(scored):
    q, cache, table, lens = _paged()
    scores = torch.zeros((2, 8, 64))

    def call(q=q, cache=cache, table=table, lens=lens, **k):
        if scored:
            return ops.decode_attention_scored(q, cache, table, lens, k.pop("scores", scores), **k)
        return ops.decode_attention_window(q, cache, table, lens, k.pop("window", 3), k.pop("sinks", 1), **k)

    _bad("current GPU", call)
    _bad("q must be", call, q=q.float())
    _bad("q must be", call, q=q[None])
    _bad("kv_cache", call, cache=cache.float())
    _bad("kv_cache", call, cache=cache[:, :, :8])
    _bad("kv_cache", call, cache=cache[:0])
    _bad("block_table", call, table=table.long())
    _bad("block_table", call, table=table[:, :0])
    _bad("row per sequence", call, table=table[:1])
    _bad("seq_lens", call, lens=lens[:1])
    _bad("seq_lens", call, lens=lens.long())
    for split in (3, 66, -2):
        _bad("split_pages", call, split_pages=split)
    for pages in (0, 5):
        _bad("max_pages", call, max_pages=pages)
    _bad("out", call, out=torch.zeros((2, 32, 128)))
    _bad("lse", call, lse=torch.zeros((2, 31)))
    if scored:
        _bad("scores", call, scores=scores[:, :, :63])
        _bad("scores", call, scores=scores.double())
        _bad("scores", call, scores=scores[:1])
        _bad("share", call, scores=torch.zeros((1, 8, 64)).expand(2, 8, 64))
        _bad("share", call, scores=torch.zeros((2, 1, 64)).expand(2, 8, 64))
    else:
        _bad("window", call, window=0)
        _bad("window", call, sinks=-1)


@pytest.mark.parametrize("scores", [False, True])
def test_chunks(scores):
    q, cache, table, _ = _paged()
    q = torch.zeros((10, 32, 128), dtype=BF)
    lse, sc = torch.zeros((10, 32)), torch.zeros((2, 8, 64))

    def call(qs, ks, q=q, **k):
        if scores:
            return ops.paged_prefill_scores(q, cache, table, qs, ks, k.get("lse", lse), k.get("scores", sc))
        return ops.paged_prefill_attention_window(q, cache, table, qs, ks, 3, 1, **k)

    _bad("current GPU", call, [0, 4, 10], [0, 3])
    _bad("q_start", call, [0, 4], [0, 3])
    _bad("q_start", call, [1, 4, 10], [0, 3])
    _bad("q_start", call, [0, 5, 4], [0, 3])
    _bad("q_start", call, [0, 4, 11], [0, 3])
    _bad("q_start", call, [[0, 4, 10]], [0, 3])
    _bad("rows must lie", call, [0, 4, 10], [0, 59])
    _bad("rows must lie", call, [0, 4, 10], [-1, 0])
    if scores:
        _bad("lse", call, [0, 4, 10], [0, 3], lse=lse[:9])
        _bad("scores", call, [0, 4, 10], [0, 3], scores=sc[:, :, :60])
    else:
        _bad("table's rows", call, [0, 1, 2, 3], [0, 0, 0])
        _bad("out", call, [0, 4, 10], [0, 3], out=torch.zeros((10, 32, 128)))


def test_evict():
    _, cache, table, lens = _paged()
    caches = [cache, cache.clone()]
    scores, positions = torch.zeros((2, 2, 8, 64)), torch.zeros((2, 2, 8, 64), dtype=I32)

    def call(caches=caches, table=table, lens=lens, scores=scores, positions=positions, tokens=lens.clone(), budget=4, sinks=1,
             recent=2, **k):
        return ops.kv_evict(caches, table, lens, scores, positions, tokens, budget, sinks, recent, **k)

    _bad("current GPU", call)
    for budget, sinks, recent in ((0, 0, 0), (4, 3, 2), (4, -1, 2), (4, 1, -1), (1 << 31, 0, 0)):
        _bad("budget", call, budget=budget, sinks=sinks, recent=recent)
    _bad("layer caches", call, caches=[], scores=scores[:0], positions=positions[:0])
    _bad("layer caches", call, caches=[cache] * 17, scores=torch.zeros(17, 2, 8, 64),
         positions=torch.zeros(17, 2, 8, 64, dtype=I32))
    _bad("layer caches", call, caches=[cache, cache[:5]])
    _bad("layer caches", call, caches=[cache.float(), cache.float()])
    _bad("scores and positions", call, scores=scores[:1])
    _bad("scores and positions", call, scores=scores[..., :63])
    _bad("scores and positions", call, positions=positions.long())
    _bad("scores and positions", call, positions=torch.zeros((2, 2, 8, 80), dtype=I32))
    _bad("seq_lens", call, lens=lens.long())
    _bad("seq_lens", call, tokens=lens[:1])
    _bad("row per sequence", call, table=table[:1])
    _bad("max_pages", call, max_pages=5)
    _bad("out", call, out=lens)
    _bad("out", call, out=torch.zeros(3, dtype=I32))


def test_c_entry_points_return_errors():
    """Bad arguments that get past no launch (the pointers are never followed)."""
    L, one = lib(), 1 << 12
    bad = 1                                                  # hipErrorInvalidValue

    def win(window=4, sinks=0, q=one):
        return L.abkv_window_attn(q, 1, 1, 1, one, 1, 1, 1, one, 1, 1, 1, 1, 8, None, window, sinks, 1.0, one, 1, 1, 1, None, None, 0)

    def scaled(scale, stride=1):
        return (L.abkv_window_attn(one, 1, stride, 1, one, 1, 1, 1, one, 1, 1, 1, 1, 8, None, 4, 0, scale, one, 1, 1, 1, None, None,
                                   0),
                L.abkv_window_attn_f32(one, 1, stride, 1, one, 1, 1, 1, one, 1, 1, 1, 1, 8, None, 4, 0, scale, one, 1, 1, 1, None,
                                       0),
                L.abkv_window_attn_bwd(one, 1, stride, 1, *[one, 1, 1, 1] * 4, one, None, 1, 8, None, 4, 0, scale,
                                       *[one, 1, 1, 1] * 3,
                                       one, 1 << 30, 0),
                L.abkv_paged_prefill_attn_window(one, stride, 1, one, 4, one, 4, 4, one, one, 1, 4, 0, scale, one, 1, 1, None, 0),
                L.abkv_paged_prefill_scores(one, stride, 1, one, 4, one, 4, 4, one, one, 1, 64, one, one, 64, 64, scale, 0))

    assert set(scaled(0.0) + scaled(-1.0) + scaled(float("nan")) + scaled(float("inf")) + scaled(1.0, 1 << 24)) == {bad}
    assert win(0) == win(4, -1) == win(q=0) == bad
    assert L.abkv_window_attn(one, 1, 1, 1, one, 1, 1, 1, one, 1, 1, 1, 0, 8, None, 4, 0, 1.0, one, 1, 1, 1, None, None, 0) == 0
    args = [one, 1, 1, 1] * 5 + [one, None, 1, 8, None, 4, 0, 1.0] + [one, 1, 1, 1] * 3
    assert L.abkv_window_attn_bwd(*args, one, 16, 0) == bad                              # workspace too small
    assert L.abkv_window_attn_bwd(*args, 0, 1 << 30, 0) == bad

    def dec(window=4, sinks=0, split=2, pages=4, seqs=1, stride=4, ws=one, size=1 << 30):
        return L.abkv_decode_attn_window(one, 1, 1, one, 4, one, stride, one, seqs, pages, split, window, sinks, 1.0, one, 1, 1,
                                         None, ws, size, 0)

    assert L.abkv_decode_attn_window(one, 1, 1, one, 4, one, 4, one, 1, 4, 2, 4, 0, 0.0, one, 1, 1, None, one, 1 << 30, 0) == bad
    assert L.abkv_decode_attn_scored(one, 1, 1, one, 4, one, 4, one, 1, 4, 2, -1.0, one, 64, 64, one, 1, 1, None, one, 1 << 30,
                                     0) == bad
    assert dec(0) == dec(4, -1) == dec(split=3) == dec(split=66) == dec(pages=0) == dec(seqs=65536) == dec(stride=3) == bad
    assert dec(window=64, size=8) == dec(window=64, ws=0) == bad
    assert dec(seqs=0) == 0
    assert L.abkv_decode_attn_scored(one, 1, 1, one, 4, one, 40, one, 1, 40, 2, 1.0, one, 640, 640, one, 1, 1, None, 0, 0,
                                     0) == bad
    assert L.abkv_decode_attn_scored(one, 1, 1, one, 4, one, 40, one, 1, 40, 2, 1.0, 0, 640, 640, one, 1, 1, None, one,
                                     1 << 30, 0) == bad
    assert L.abkv_paged_prefill_scores(one, 1, 1, one, 4, one, 4, 4, one, one, 1, 96, one, one, 64, 64, 1.0, 0) == bad

    def chunk(starts, past, requests=None, width=4):
        starts, past = (C.c_int32 * len(starts))(*starts), (C.c_int32 * len(past))(*past)
        batch = (one, 4096, 128, one, 4, one, width, width, C.addressof(starts), C.addressof(past),
                 len(past) if requests is None else requests)
        rc = L.abkv_paged_prefill_attn_window(*batch, 4, 0, 1.0, one, 4096, 128, None, 0)
        assert rc == L.abkv_paged_prefill_scores(*batch, 64, one, one, 512, 64, 1.0, 0)
        return rc

    assert chunk([0, 1], [64]) == chunk([0, 65], [0]) == chunk([2, 1], [0]) == chunk([0, 1], [-1]) == chunk([-1, 0], [0]) == bad
    assert chunk([0, 1, 2], [0, 64]) == bad and chunk([0, 5], [0], 0) == chunk([3, 3, 3], [0, 64]) == 0     # nothing to launch
    caches = (C.c_void_p * 1)(one)

    def ev(layers=1, budget=4, sinks=0, recent=0, pages=4, rows=64, arr=caches, ws=None):
        return L.abkv_kv_evict(arr, layers, 4, one, 1 << 20, one, 1, pages, one, one, rows, one, budget, sinks, recent, one, ws,
                               0, 0)

    assert ev(17) == ev(budget=0) == ev(budget=4, sinks=3, recent=2) == ev(pages=0) == ev(rows=63) == bad
    assert ev(pages=16385, rows=1 << 20) == ev(pages=4000, rows=64000) == bad             # too long; without its workspace
    assert ev(arr=(C.c_void_p * 1)(None)) == bad and ev(0) == 0


def test_backend_and_model_options():
    with pytest.raises(ValueError, match="sinks"):
        bk.AbridgeAttentionImpl(sinks=4)
    for window, sinks in ((0, 0), (-3, 0), (4, -1)):
        with pytest.raises(ValueError):
            bk.AbridgeAttentionImpl(sliding_window=window, sinks=sinks)
    impl = bk.AbridgeAttentionImpl(sliding_window=64, sinks=4)
    md = bk.AbridgeAttentionMetadata(np.array([0, 4]), np.array([8]), None, None, None, 0, np.array([6]), 1)
    with pytest.raises(NotImplementedError, match="causal"):
        impl.attend(None, None, md, None)


def test_attention_function_masks():
    import types

    from abridgekv_amd.compress_forward import CompressMask, WindowMask, masked_attention_forward
    q, k, v = (t.transpose(1, 2) for t in _dense())
    module = types.SimpleNamespace(layer_idx=0)
    with pytest.raises(NotImplementedError, match="sliding"):
        masked_attention_forward(module, q, k, v, CompressMask(9, 0, 1), sliding_window=4)
    with pytest.raises(NotImplementedError, match="sliding"):
        masked_attention_forward(module, q, k, v, WindowMask(4), sliding_window=4)
    with pytest.raises(TypeError):
        masked_attention_forward(module, q, k, v, torch.ones(2))
    with pytest.raises(NotImplementedError, match="dropout"):
        masked_attention_forward(module, q, k, v, WindowMask(4), dropout=0.1)
    with pytest.raises(ValueError, match="current GPU"):
        masked_attention_forward(module, q, k, v, None, sliding_window=4)
    qf = q.float().requires_grad_(True)
    with pytest.raises(NotImplementedError, match="bf16"):
        masked_attention_forward(module, qf, k.float(), v.float(), WindowMask(4))


def test_step_splits():
    """Every split choice is valid, covers the pages and leaves a workspace that holds it."""
    for seqs in (1, 3, 24, 64, 300, 65535):
        for pages in (1, 2, 3, 15, 28, 29, 64, 160, 257, 2049, 16384):
            sp = ops._step_split_pages(seqs, pages)
            assert 2 <= sp <= 64 and sp % 2 == 0, (seqs, pages, sp)
            for window, sinks in ((1, 0), (100, 4), (4096, 300), ((1 << 31) - 1, (1 << 31) - 1)):
                sp = ops.window_split_pages(seqs, pages, window, sinks)
                assert 2 <= sp <= 64 and sp % 2 == 0, (seqs, pages, window, sinks, sp)
                need = min(pages, -(-sinks // 16) - (-window // 16) + 1)
                if need <= 28:
                    assert ops.decode_window_bytes(seqs, pages, window, sinks, sp) == 0


def test_score_tiles():
    for ks, nq in (([0], [1]), ([0, 500], [2048, 3]), ([8000], [64]), ([7, 0], [0, 2])):
        assert ops._score_tile_keys(np.array(ks), np.array(nq), 256) in (64, 128)
