"""What the fused norms, the 4-bit cache and the log probabilities refuse, on the CPU: every bad argument is named before any
launch, and good ones get as far as the device check. The C entry points return an error code for theirs."""
import types

import pytest
import torch

from abridgekv_amd import backend as bk
from abridgekv_amd import fused, ops
from abridgekv_amd._lib import lib

BF, F32, I32, I64 = torch.bfloat16, torch.float32, torch.int32, torch.int64
GPU = "current GPU"


def _bad(match, call, *a, **k):
    with pytest.raises(ValueError, match=match):
        call(*a, **k)


def _cache(pages=4):
    return torch.zeros(ops.kv_cache_int4_shape(pages), dtype=torch.uint8)


def _kv(T=3):
    return torch.zeros((T, 8, 128), dtype=BF), torch.zeros((T, 8, 128), dtype=BF), torch.zeros(T, dtype=I64)


BAD_CACHES = [torch.zeros(ops.kv_cache_shape(4), dtype=BF), torch.zeros((4, 2, 16, 641), dtype=torch.uint8),
              torch.zeros((0, 2, 16, 640), dtype=torch.uint8), torch.zeros((4, 2, 16, 1280), dtype=torch.uint8)[..., ::2],
              torch.zeros((8, 2, 16, 640), dtype=torch.uint8)[::2], torch.zeros(4 * 20480 + 1, dtype=torch.uint8)[1:].view(4, 2, 16, 640)]


def test_append_and_read():
    k, v, s = _kv()
    _bad(GPU, ops.kv_append_int4, k, v, s, _cache())
    for bad in BAD_CACHES:
        _bad("kv_cache", ops.kv_append_int4, k, v, s, bad)
        _bad("kv_cache", ops.kv_read_int4, bad, s)
    _bad("key must be", ops.kv_append_int4, k.float(), v, s, _cache())
    _bad("key must be", ops.kv_append_int4, k[:2], v, s, _cache())
    _bad("value must", ops.kv_append_int4, k, torch.zeros((3, 8, 132), dtype=BF)[..., :128], s, _cache())
    _bad("value must", ops.kv_append_int4, k, torch.zeros((3, 128, 8), dtype=BF).transpose(1, 2), s, _cache())
    _bad("slot_mapping", ops.kv_append_int4, k, v, s.int(), _cache())
    _bad("slot_mapping", ops.kv_append_int4, k, v, torch.zeros(6, dtype=I64)[::2], _cache())
    _bad(GPU, ops.kv_read_int4, _cache(), s)
    _bad("float32 or bfloat16", ops.kv_read_int4, _cache(), s, torch.float16)


def _step(B=2):
    return (torch.zeros((B, 32, 128), dtype=BF), _cache(), torch.zeros((B, 4), dtype=I32), torch.zeros(B, dtype=I32))


def test_decode():
    q, c, t, n = _step()
    _bad(GPU, ops.decode_attention_int4, q, c, t, n)
    for bad in BAD_CACHES:
        _bad("kv_cache", ops.decode_attention_int4, q, bad, t, n)
    _bad("q must be", ops.decode_attention_int4, q.float(), c, t, n)
    _bad("q must be", ops.decode_attention_int4, q[:, :8], c, t, n)
    _bad("block_table", ops.decode_attention_int4, q, c, t[:1], n)
    _bad("block_table", ops.decode_attention_int4, q, c, t.long(), n)
    _bad("seq_lens", ops.decode_attention_int4, q, c, t, n[:1])
    _bad("seq_lens", ops.decode_attention_int4, q, c, t, n.long())
    for pages in (0, 5):
        _bad("max_pages", ops.decode_attention_int4, q, c, t, n, max_pages=pages)
    for split in (3, 66, -2):
        _bad("split_pages", ops.decode_attention_int4, q, c, t, n, split_pages=split)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        _bad("scale", ops.decode_attention_int4, q, c, t, n, scale=scale)
    _bad("out must be", ops.decode_attention_int4, q, c, t, n, out=q.float())
    _bad("share memory", ops.decode_attention_int4, q, c, t, n, out=q[:1].expand(2, -1, -1))
    _bad("lse", ops.decode_attention_int4, q, c, t, n, lse=torch.zeros(2, 31))


def test_chunks():
    q, c, t, _ = _step(5)
    args = ([0, 3, 5], [4, 0], [7, 2], True)
    _bad(GPU, ops.paged_prefill_attention_int4, q, c, t, *args)
    for bad in BAD_CACHES:
        _bad("kv_cache", ops.paged_prefill_attention_int4, q, bad, t, *args)
    _bad("q must be", ops.paged_prefill_attention_int4, q.float(), c, t, *args)
    _bad("block_table", ops.paged_prefill_attention_int4, q, c, t.long(), *args)
    _bad("kv_limit", ops.paged_prefill_attention_int4, q, c, t, [0, 3, 5], [4, 0], [7, 65], True)
    _bad("kv_limit", ops.paged_prefill_attention_int4, q, c, t, [0, 3, 5], [4, 0], [-1, 2], True)
    _bad("scale", ops.paged_prefill_attention_int4, q, c, t, *args, scale=-1.0)


def _append(T=3, **kw):
    k, v, s = _kv(T)
    base = dict(q=torch.zeros((T, 32, 128), dtype=BF), key=k, value=v, positions=torch.zeros(T, dtype=I64),
                cos_sin=torch.zeros(9, 128), slot_mapping=s, kv_cache=torch.zeros(ops.kv_cache_shape(2), dtype=BF),
                q_weight=torch.zeros(128, dtype=BF), k_weight=torch.zeros(128, dtype=BF), max_position=8)
    base.update(kw)
    return lambda: ops.qk_norm_rope_append(**base)


def test_norm_append():
    _bad(GPU, _append())
    _bad(GPU, _append(kv_cache=_cache(), q_weight=None, k_weight=None))
    _bad("q must be", _append(q=torch.zeros((3, 32, 128))))
    _bad("key must be", _append(key=torch.zeros((2, 8, 128), dtype=BF)))
    _bad("value must", _append(value=torch.zeros((3, 8, 129), dtype=BF)[..., 1:]))
    _bad("positions", _append(positions=torch.zeros(3, dtype=I32)))
    _bad("cos_sin", _append(cos_sin=torch.zeros(9, 64)))
    _bad("cos_sin", _append(cos_sin=torch.zeros(9, 128, dtype=BF)))
    _bad("slot_mapping", _append(slot_mapping=torch.zeros(4, dtype=I64)))
    _bad("kv_cache", _append(kv_cache=torch.zeros((2, 2, 16, 600), dtype=torch.uint8)))
    with pytest.raises(ValueError):
        _append(kv_cache=torch.zeros(ops.kv_cache_shape(2)))()
    _bad("neither", _append(q_weight=None))
    _bad("weight", _append(q_weight=torch.zeros(64, dtype=BF)))
    _bad("weight", _append(k_weight=torch.zeros(128, dtype=torch.float16)))
    _bad("one type", _append(k_weight=torch.zeros(128)))
    for eps in (-1e-6, float("nan"), float("inf")):
        _bad("eps", _append(eps=eps))
    _bad("codes_k", _append(block_c=64, codes_k=12))
    _bad("code_span", _append(block_c=64, codes_k=16, code_span=65))
    _bad("out must", _append(out=torch.zeros((3, 32, 128))))


def _train(B=2, S=3, dt=BF):
    q, k = torch.zeros((B, S, 32, 128), dtype=dt), torch.zeros((B, S, 8, 128), dtype=dt)
    return q, k, torch.zeros((1, S, 128), dtype=dt), torch.zeros((1, S, 128), dtype=dt), torch.ones(128, dtype=dt), torch.ones(128, dtype=dt)


def test_norm_training():
    q, k, c, s, wq, wk = _train()
    for call in (ops.qk_norm_rope, fused.qk_norm_rope):
        _bad(GPU, call, q, k, c, s, wq, wk)
        _bad("q must be", call, q.half(), k, c, s, wq, wk)
        _bad("q must be", call, q[0], k, c, s, wq, wk)
        _bad("k must be", call, q, k.float(), c, s, wq, wk)
        _bad("k must be", call, q, k[:, :2], c, s, wq, wk)
        _bad("cos must be", call, q, k, c[0], s, wq, wk)
        _bad("cos must be", call, q, k, c.expand(3, -1, -1), s, wq, wk)
        _bad("sin must be", call, q, k, c, s.float(), wq, wk)
        _bad("sin must be", call, q, k, c, s[:, :2], wq, wk)
        _bad("weight", call, q, k, c, s, wq[:64], wk)
        _bad("one type", call, q, k, c, s, wq.float(), wk)
        _bad("eps", call, q, k, c, s, wq, wk, -1.0)
    _bad(GPU, ops.qk_norm_rope_backward, q, k, q, k, c, s, wq, wk)
    _bad("dq_out", ops.qk_norm_rope_backward, q, k, k, k, c, s, wq, wk)
    _bad("dk_out", ops.qk_norm_rope_backward, q, k, q, k.float(), c, s, wq, wk)
    with pytest.raises(NotImplementedError, match="angles"):
        fused.qk_norm_rope(q, k, c.requires_grad_(True), s, wq, wk)


def test_head_norms():
    norm = types.SimpleNamespace(weight=torch.ones(128), variance_epsilon=1e-6)
    wide = types.SimpleNamespace(weight=torch.ones(4096), variance_epsilon=1e-6)
    assert fused.head_norms(types.SimpleNamespace()) == (None, None, 0.0)
    assert fused.head_norms(types.SimpleNamespace(q_norm=norm, k_norm=norm))[2] == 1e-6
    other = types.SimpleNamespace(weight=torch.ones(128), variance_epsilon=1e-5)
    for q, k in ((norm, None), (wide, wide), (norm, other), (types.SimpleNamespace(weight=torch.ones(128)), norm)):
        with pytest.raises(NotImplementedError, match="norms"):
            fused.head_norms(types.SimpleNamespace(q_norm=q, k_norm=k))


def test_logprobs():
    x, t = torch.zeros((3, 50)), torch.zeros(3, dtype=I64)
    for call in (ops.token_logprobs, fused.token_logprobs):
        _bad(GPU, call, x, t)
        _bad("logits", call, x.double(), t)
        _bad("logits", call, x[0], t)
        _bad("logits", call, x.T, t)
        _bad("logits", call, x[:, :0], t)
        _bad("logits", call, x[:1].expand(3, -1), t)
        _bad("targets", call, x, t.int())
        _bad("targets", call, x, t[:2])
        for temperature in (0.0, -1.0, float("nan"), float("inf")):
            _bad("temperature", call, x, t, temperature)
    for top in (-1, 33):
        _bad("top", ops.token_logprobs, x, t, top=top)
    _bad("top", ops.token_logprobs, x[:, :4], t, top=5)
    st, g = torch.zeros((3, 3)), torch.zeros(3)
    _bad(GPU, ops.token_logprobs_backward, x, t, st, g)
    _bad("stats", ops.token_logprobs_backward, x, t, st[:2], g)
    _bad("dlogprob", ops.token_logprobs_backward, x, t, st, g.double())
    _bad("dentropy", ops.token_logprobs_backward, x, t, st, None, g[:2])
    _bad("out must", ops.token_logprobs_backward, x, t, st, g, out=x.to(BF))
    _bad("out must", ops.token_logprobs_backward, x, t, st, g, out=x[:1].expand(3, -1))


def test_moves_take_one_kind_of_cache():
    a, b = _cache(), torch.zeros(ops.kv_cache_shape(4), dtype=BF)
    with pytest.raises(ValueError, match="one kind"):
        ops._row_geometry([a, b])
    assert ops._row_geometry([a, a]) == (16, 20480, 10240, 640)


def test_backend():
    with pytest.raises(NotImplementedError, match="dtype"):
        bk.AbridgeAttentionImpl(kv_cache_dtype="fp8")
    with pytest.raises(NotImplementedError, match="sliding window"):
        bk.AbridgeAttentionImpl(kv_cache_dtype="int4", sliding_window=64)
    assert bk.AbridgeAttentionBackend.get_kv_cache_shape(7, kv_cache_dtype="int4") == (7, 2, 16, 640)
    assert bk.AbridgeAttentionBackend.get_kv_cache_shape(7) == (7, 2, 16, 8, 128)


def test_c_entries_return_errors():
    """Null and misaligned pointers, sizes out of range: an error code, and nothing launched."""
    L = lib()
    p = torch.zeros(1 << 16, dtype=torch.uint8)
    a = p.data_ptr() + (-p.data_ptr()) % 16
    assert L.abkv_kv_append_int4(None, 1024, 128, a, 1024, 128, a, 1, a, 1, None) != 0
    assert L.abkv_kv_append_int4(a + 2, 1024, 128, a, 1024, 128, a, 1, a, 1, None) != 0
    assert L.abkv_kv_append_int4(a, 1024, 130, a, 1024, 128, a, 1, a, 1, None) != 0
    assert L.abkv_kv_append_int4(a, 1024, 128, a, 1024, 128, a, 0, a, 1, None) == 0
    assert L.abkv_kv_read_int4(a, 0, a, 1, 1, a, a, None) != 0
    dec = [a, 4096, 128, a, 1, a, 4, a, 1, 4, 2, 0.1, a, 4096, 128, None, a, 1 << 20, None]
    for i, bad in ((0, None), (3, None), (4, 0), (6, 3), (10, 3), (10, 66), (11, -1.0), (16, None), (17, 100), (8, 70000), (0, a + 2)):
        assert L.abkv_decode_attn_int4(*dec[:i], bad, *dec[i + 1:]) != 0, i
    pre = [a, 4096, 128, a, 1, a, 4, 4, a, a, a, None, a, a, 1, a, 0, 0, 0.1, a, 4096, 128, None, a, 1 << 20, None]
    for i, bad in ((0, None), (0, a + 2), (1, 4097), (3, None), (3, a + 8), (4, 0), (5, None), (7, 0), (12, None), (16, -1), (17, 64),
                   (18, -1.0), (18, float("inf")), (19, a + 8), (20, 4100)):
        assert L.abkv_paged_prefill_attn_items_int4(*pre[:i], bad, *pre[i + 1:]) != 0, i
    app = [a, 4096, 128, a, 1024, 128, a, 1024, 128, a, 1, a, a, 0, 1e-6, 0, 0, 0, a, 9, a, a, 1, 0, a, 4096, 128, None]
    for i, bad in ((0, None), (0, a + 4), (4, 1020), (9, None), (11, None), (14, -1.0), (15, -1), (19, 0), (20, None), (22, 0),
                   (24, None)):
        assert L.abkv_qk_norm_rope_append(*app[:i], bad, *app[i + 1:]) != 0, i
    tr = [0, a, 8192, 4096, 128, a, 2048, 1024, 128, 1, 2, a, a, 0, 1e-6, a, a, 0, 128, 0, a, a, None]
    for i, bad in ((1, None), (3, 4097), (5, None), (11, None), (12, a + 2), (14, -1.0), (15, None), (18, 130), (20, None)):
        assert L.abkv_qk_norm_rope(*tr[:i], bad, *tr[i + 1:]) != 0, i
    lp = [0, a, 50, 2, 50, a, 1.0, 0, a, a, a, a, a, a, 1 << 20, None]
    for i, bad in ((1, None), (1, a + 1), (2, 40), (4, 0), (5, None), (6, 0.0), (7, 33), (7, 51), (8, None), (14, 3)):
        assert L.abkv_token_logprobs(*lp[:i], bad, *lp[i + 1:]) != 0, i
    assert L.abkv_token_logprobs(*lp[:7], 3, *lp[8:11], None, *lp[12:]) != 0
    bw = [0, a, 50, 2, 50, a, 1.0, a, a, a, a, 50, None]
    for i, bad in ((1, None), (2, 49), (4, -1), (6, -1.0), (7, None), (10, None), (10, a + 1), (11, 49)):
        assert L.abkv_token_logprobs_bwd(*bw[:i], bad, *bw[i + 1:]) != 0, i
    assert L.abkv_qk_norm_rope_bwd_workspace_size(0, 5) == 0 and L.abkv_qk_norm_rope_bwd_workspace_size(2, 5) > 0
    assert L.abkv_decode_int4_workspace_size(2, 4, 4) == 0
    assert L.abkv_decode_int4_workspace_size(2, 4, 2) == 2 * 2 * 32 * (256 + 16)


def test_int4_splits_fit_any_step():
    """Equal shares or an even number of pages up to 64; a step of shorter tables and fewer sequences finds room in what a builder
    holds for the longest ones: its own splits or shares, or longer splits."""
    for most in (1, 2, 64, 512, 520):
        for longest in (1, 3, 65, 129, 512, 513, 8191, 8193, 40000):
            held = max(ops.decode_int4_bytes(b, longest, ops.int4_split_pages(b, longest)) for b in range(1, most + 1))
            for b in {1, most // 2 + 1, most}:
                for pages in {1, longest // 3 + 1, longest - 1 or 1, longest}:
                    split = ops.int4_split_pages(b, pages)
                    assert split % 2 == 0 and 0 <= split <= 64 and (split > 0 or (b <= 512 and b * pages > 8192))
                    need = ops.decode_int4_bytes(b, pages, split)
                    assert need <= held or (split > 0 and ops.decode_int4_bytes(b, pages, 64) <= held)
    q, c = torch.zeros((513, 32, 128), dtype=BF), _cache()
    _bad("512 sequences", ops.decode_attention_int4, q, c, torch.zeros((513, 4), dtype=I32), torch.zeros(513, dtype=I32), split_pages=0)
