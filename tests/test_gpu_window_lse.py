"""The log-sum-exp of attention under a sliding window, where a few keys weigh far more than those before them. The running
maximum of the softmax moves only past a headroom of 2^8, so weights up to 256 are summed; each of them rounded to bf16 would
leave lse up to 2^-8 off however many rows are visible."""
import numpy as np
import pytest
import torch

from oracle import window as ow

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5
LOG2E = 1.4426950408889634
E32 = 2.0 ** -24


def _peaked(seed, S, peaks):
    """bf16 q [S, 32, 128], k, v [S, 8, 128]: key t of ``peaks`` scores about peaks[t] log2 units above the flat ones."""
    gen = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn((S, h, 128), generator=gen) * s for h, s in ((32, 0.5), (8, 0.5), (8, 1.0)))
    q[..., 0], k[..., 0] = 8.0, 0.0
    for t, up in peaks.items():
        k[t, :, 0] = up / (8 * SCALE * LOG2E)
    return q.to(torch.bfloat16), k.to(torch.bfloat16), v.to(torch.bfloat16)


def _bound(q, k, lse):
    """fp32 arithmetic: a score's 128 products summed in any order (128 half steps of the sum of |q k|) and scaled, its distance
    to the maximum (two operations on values below 64), an exponential and a logarithm good to a step, and up to S weights
    summed (S half steps)."""
    q, k = q.double().abs().numpy(), np.repeat(k.double().abs().numpy(), 4, 1)
    most = SCALE * np.einsum("ihd,jhd->hij", q, k).max()
    return 1.02 * (E32 * (128 * most + 4 * 64 + 8 + q.shape[0]) + E32 * np.abs(lse[np.isfinite(lse)]).max())


PEAKS = [{100: 3.1}, {100: 4.7, 300: 7.3}, {70: 6.6}, {2: 5.9}, {1: 3.3, 200: 6.1, 450: 7.7}, {0: 7.9, 63: 7.2}]


@pytest.mark.parametrize("peaks", PEAKS)
@pytest.mark.parametrize("window,sinks", [(1000, 0), (256, 4), (200, 70)])
def test_prompts(peaks, window, sinks):
    from abridgekv_amd import ops
    S = 600
    q, k, v = _peaked(S + window, S, peaks)
    vis = ow.visible(np.arange(S), S, window, sinks)
    _, want, _ = ow.attend(q.double().numpy(), k.double().numpy(), v.double().numpy(), vis, SCALE)
    lse, low_lse = (torch.empty((1, 32, S), device="cuda") for _ in range(2))
    qkv = [t[None].cuda() for t in (q, k, v)]
    out, _ = ops.window_attention(*qkv, window, sinks, lse=lse)
    low = torch.empty((1, S, 32, 128), dtype=torch.float8_e5m2, device="cuda")
    ops.window_attention(*qkv, window, sinks, lse=low_lse, out_low=low)
    assert torch.equal(lse, low_lse)
    assert torch.equal(out, ops.window_attention(*qkv, window, sinks)[0])
    err = np.abs(lse[0].double().cpu().numpy().T - want).max()
    assert err <= _bound(q, k, want), (err, _bound(q, k, want))


@pytest.mark.parametrize("peaks", PEAKS)
@pytest.mark.parametrize("window,sinks", [(1000, 0), (256, 4), (200, 70)])
def test_chunks(peaks, window, sinks):
    from abridgekv_amd import ops
    S, past = 600, 470
    q, k, v = _peaked(S + window, S, peaks)
    vis = ow.visible(np.arange(past, S), S, window, sinks)
    _, want, _ = ow.attend(q[past:].double().numpy(), k.double().numpy(), v.double().numpy(), vis, SCALE)
    cache = torch.zeros((38, 2, 16, 8, 128), dtype=torch.bfloat16)
    at = torch.arange(S)
    for i, rows in enumerate((k, v)):
        cache[at // 16, i, at % 16] = rows
    table = torch.arange(38, dtype=torch.int32)[None].cuda()
    lse = torch.empty((S - past, 32), device="cuda")
    ops.paged_prefill_attention_window(q[past:].cuda(), cache.cuda(), table, [0, S - past], [past], window, sinks, lse=lse)
    err = np.abs(lse.double().cpu().numpy() - want).max()
    assert err <= _bound(q, k, want), (err, _bound(q, k, want))


@pytest.mark.parametrize("peaks", PEAKS[:4])
def test_gradients(peaks):
    """Under that lse, within the oracle's bounds element by element."""
    from abridgekv_amd import ops
    S, window, sinks = 400, 256, 4
    q, k, v = (t[None] for t in _peaked(S, S, peaks))
    g = torch.randn((1, S, 32, 128), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    dev = [t.cuda() for t in (q, k, v)]
    lse = torch.empty((1, 32, S), device="cuda")
    low = torch.empty((1, S, 32, 128), dtype=torch.float8_e5m2, device="cuda")
    out, _ = ops.window_attention(*dev, window, sinks, lse=lse, out_low=low)
    got = ops.window_attention_backward(*dev, out, lse, g.cuda(), window, sinks, out_low=low)
    want = ow.window_backward(*(t.double().numpy() for t in (q, k, v, g)), None, window, sinks, SCALE, bounds=True)
    for name, x, d, tol in zip(("dq", "dk", "dv"), got, want[::2], want[1::2]):
        assert (np.abs(x.double().cpu().numpy() - d) <= tol).all(), name
