"""Prompt chunks under a sliding window read no row that the chunk does not see: rows between the sinks and the first query's
window may hold anything, and the table's entries of pages that lie between them may be any number."""
import numpy as np
import pytest
import torch

from abridgekv_amd import backend as bk
from abridgekv_amd import ops

pytestmark = pytest.mark.gpu

CHUNK, PAST = [1, 64, 130, 33, 70, 200], [500, 300, 640, 777, 64, 1000]


def _batch(seed, chunk=CHUNK, past=PAST):
    """A cache of finite rows over scattered pages, its table, and queries."""
    gen = torch.Generator().manual_seed(seed)
    need = [-(-(c + p) // 16) for c, p in zip(chunk, past)]
    pool = sum(need) + 3
    pages = np.random.default_rng(seed).permutation(pool)[: sum(need)]
    table = np.zeros((len(need), max(need)), np.int32)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = pages[at: at + n]
        at += n
    cache = torch.randn((pool, 2, 16, 8, 128), generator=gen).to(torch.bfloat16)
    q = torch.randn((sum(chunk), 32, 128), generator=gen).to(torch.bfloat16)
    return q, cache, table


def _hide(cache, table, window, sinks, value, ids, past=PAST):
    """The rows that no query of a request sees hold ``value``; the table's entries of pages wholly among them become ``ids``
    where that is a number."""
    cache, table = cache.clone(), table.copy()
    for r, p in enumerate(past):
        rows = np.arange(min(sinks, p), max(p + 1 - window, 0))
        cache[torch.from_numpy(table[r, rows // 16].astype(np.int64)), :, torch.from_numpy(rows % 16)] = value
        if ids is not None and rows.size:
            table[r, -(-rows[0] // 16): (rows[-1] + 1) // 16] = ids
    return cache, table


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (40, 4), (64, 16), (63, 17), (100, 32), (100, 33), (129, 64), (200, 70),
                                          (300, 130)])
@pytest.mark.parametrize("value,ids", [(float("nan"), None), (float("inf"), 1 << 30), (float("-inf"), -7)])
def test_hidden_rows_may_hold_anything(window, sinks, value, ids):
    q, cache, table = _batch(window + sinks)
    q_start = np.concatenate([[0], np.cumsum(CHUNK)])
    q = q.cuda()
    lse, want_lse = (torch.empty((q.shape[0], 32), device="cuda") for _ in range(2))
    want, _ = ops.paged_prefill_attention_window(q, cache.cuda(), torch.from_numpy(table).cuda(), q_start, PAST, window, sinks,
                                                 lse=want_lse)
    bad, ids_table = _hide(cache, table, window, sinks, value, ids)
    got, _ = ops.paged_prefill_attention_window(q, bad.cuda(), torch.from_numpy(ids_table).cuda(), q_start, PAST, window, sinks,
                                                lse=lse)
    assert torch.isfinite(want).all() and torch.isfinite(want_lse).all()
    assert torch.equal(got, want) and torch.equal(lse, want_lse)


def test_backend_layer_with_pages_given_back():
    """A windowed layer's step of two decodes and two chunks, the pages outside the windows taken away."""
    qlen, past, window, sinks = [1, 1, 90, 64], [640, 200, 500, 333], 100, 4
    q, cache, table = _batch(3, qlen, past)
    seq = [c + p for c, p in zip(qlen, past)]
    T = sum(qlen)
    gen = torch.Generator().manual_seed(4)
    k, v = (torch.randn((T, 8 * 128), generator=gen).to(torch.bfloat16).cuda() for _ in range(2))
    pos = np.concatenate([np.arange(n - m, n) for n, m in zip(seq, qlen)])
    impl = bk.AbridgeAttentionImpl(sliding_window=window, sinks=sinks)

    def step(c, t):
        builder = bk.AbridgeMetadataBuilder(max_num_seqs=8, max_pages=60)
        md = builder.build(np.concatenate([[0], np.cumsum(qlen)]), seq, torch.from_numpy(t).cuda(),
                           positions=torch.from_numpy(pos).cuda())
        return impl.forward(None, q.view(T, -1).cuda(), k, v, c.cuda(), md)

    want = step(cache, table)
    got = step(*_hide(cache, table, window, sinks, float("nan"), 1 << 30, past))
    assert torch.isfinite(want).all() and torch.equal(got, want)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (40, 4), (63, 17), (100, 32), (300, 130), (700, 5)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("split_pages", [None, 2])
def test_hidden_rows_of_a_decode_step(window, sinks, value, split_pages):
    """Those on the edge pages of the sinks and of the window, and the rows past the sequence, among them."""
    past = [0, 40, 299, 640, 1000]
    q, cache, table = _batch(window, [1] * 5, past)
    bad, ids_table = _hide(cache, table, window, sinks, value, 1 << 30, past)
    for r, p in enumerate(past):                             # (the rest of the last page)
        bad[int(table[r, p // 16]), :, p % 16 + 1:] = value
    lens = torch.tensor([p + 1 for p in past], dtype=torch.int32, device="cuda")
    got = []
    for c, t in ((cache, table), (bad, ids_table)):
        lse = torch.empty((5, 32), device="cuda")
        out, _ = ops.decode_attention_window(q.cuda(), c.cuda(), torch.from_numpy(t).cuda(), lens, window, sinks, lse=lse,
                                             split_pages=split_pages)
        assert torch.isfinite(out).all() and torch.isfinite(lse).all()
        got.append((out, lse))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
