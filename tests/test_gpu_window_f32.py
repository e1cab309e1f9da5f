"""The fp32 mode of attention under a sliding window: rows that are not finite reach only the rows that see them."""
import numpy as np
import pytest
import torch

from oracle import window as ow

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


@pytest.mark.parametrize("window,sinks", [(1, 0), (40, 4), (17, 33), (300, 0)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("side", ["k", "v", "both"])
def test_infinite_rows_reach_only_the_rows_that_see_them(window, sinks, bad, side):
    """Bounds as the finite inputs': 3e-5 (128-term products and sums of up to S rows in fp32, |out| <= max|v| of about 4.5)."""
    from abridgekv_amd import ops
    S, lens, at = 260, [260, 201], [(0, 97, 3), (0, 98, 3), (1, 16, 0), (1, 150, 7), (1, 1, 5)]
    gen = torch.Generator().manual_seed(window)
    q, k, v = (torch.randn((2, S, h, 128), generator=gen) for h in (32, 8, 8))
    want, want_lse = ow.window_attention(*(t.double().numpy() for t in (q, k, v)), lens, window, sinks, SCALE)
    touched = np.zeros((2, S, 32), bool)                     # output rows that see a bad one
    for b, row, h in at:
        if side != "v":
            k[b, row, h, 7] = bad
        if side != "k":
            v[b, row, h, 100:] = bad
        i = np.arange(S)
        sees = (i >= row) & ((i - row < window) | (row < sinks)) & (i < lens[b])
        touched[b, :, 4 * h: 4 * h + 4] |= sees[:, None]
    lse = torch.empty((2, 32, S), device="cuda")
    out, _ = ops.window_attention(q.cuda(), k.cuda(), v.cuda(), window, sinks, lse=lse,
                                  seq_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy().transpose(0, 2, 1)
    assert np.abs(out[~touched] - want[~touched]).max() <= 3e-5
    want_lse = want_lse.transpose(0, 2, 1)
    whole = ~touched & np.isfinite(want_lse)
    assert np.abs(lse[whole] - want_lse[whole]).max() <= 1e-5
    assert (lse[~touched & ~np.isfinite(want_lse)] == -np.inf).all()
    if side == "v":                                          # their scores are finite, the dims before 100 too
        assert np.abs(out - want)[..., :100].max() <= 3e-5
        seen = np.where(np.repeat(touched[..., None], 28, -1), out[..., 100:], np.nan)
        assert not np.isfinite(seen).any()
