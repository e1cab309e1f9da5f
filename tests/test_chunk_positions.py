"""Positions of window chunks whose count of rows would pass 32 bits are refused by both entries."""
import ctypes as C

import pytest

from abridgekv_amd._lib import lib


@pytest.mark.parametrize("start,queries", [((1 << 31) - 1, 1), ((1 << 31) - 100, 100), ((1 << 30) - 5, 6), (0, (1 << 30) + 1)])
def test_far_positions(start, queries):
    one, bad, width = 1 << 12, 1, 1 << 28                    # (a table that holds such positions)
    starts, past = (C.c_int32 * 2)(0, queries), (C.c_int32 * 1)(start)
    batch = (one, 4096, 128, one, 4, one, width, width, C.addressof(starts), C.addressof(past), 1)
    assert lib().abkv_paged_prefill_attn_window(*batch, 4, 0, 1.0, one, 4096, 128, None, 0) == bad
    assert lib().abkv_paged_prefill_scores(*batch, 64, one, one, 512, 64, 1.0, 0) == bad


@pytest.mark.parametrize("scores", [False, True])
def test_far_positions_through_ops(scores):
    import torch

    from abridgekv_amd import ops
    q, cache = torch.zeros((10, 32, 128), dtype=torch.bfloat16), torch.zeros((2, 2, 16, 8, 128), dtype=torch.bfloat16)
    table = torch.empty((1, 1 << 27), dtype=torch.int32)     # (not touched)
    wide = torch.empty((1, 8, 1 << 31), dtype=torch.float32, device="meta")
    for start, match in (((1 << 30) - 10, "current GPU"), ((1 << 30) - 9, "rows must lie"), ((1 << 31) - 10, "rows must lie")):
        with pytest.raises(ValueError, match=match):
            if scores:
                ops.paged_prefill_scores(q, cache, table, [0, 10], [start], torch.zeros(10, 32), wide)
            else:
                ops.paged_prefill_attention_window(q, cache, table, [0, 10], [start], 4)
