"""Multi-query attention over a cache in 4 bits where the softmax and the magnitudes reach far: one row that takes most of the weight,
tiny queries beside huge keys, rows that read as NaN. Against the float64 oracle."""
import numpy as np
import pytest
import torch

from oracle import int4 as oi

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


def _cache(k_rows, v_rows):
    """The rows of one sequence on pages 0, 1, ..., and its table."""
    n = len(k_rows)
    pages = -(-n // 16)
    cache = np.zeros((pages, 2, 16, 640), np.uint8)
    at = np.arange(n)
    cache[at // 16, 0, at % 16], cache[at // 16, 1, at % 16] = k_rows, v_rows
    return torch.from_numpy(cache).cuda(), torch.arange(pages, dtype=torch.int32, device="cuda")[None]


@pytest.mark.parametrize("n", [8000, 32000])
@pytest.mark.parametrize("octaves", [17, 21.6, 25.2])
@pytest.mark.parametrize("spread", [0.0, 1.0])
@pytest.mark.parametrize("at", [0, -9])
def test_one_row_far_above_the_rest(n, octaves, spread, at):
    """A row without value of its own whose weight is 2^octaves of any other's, first or near the end: what the rest leaves is the
    whole output, however little it weighs. A weight below 2^-25 of the largest is off by up to 2^-36 of that. 64 requests of two
    queries over the same rows, so that no key range is split and one walk takes them all."""
    from abridgekv_amd import ops
    B, nq = 64, 2
    gen = torch.Generator().manual_seed(n)
    k = torch.randn((n, 8, 128), generator=gen) * spread
    v = torch.randn((n, 8, 128), generator=gen) + 0.5
    q = torch.randn((B * nq, 32, 128), generator=gen)
    q[..., 5] = 4.0
    k[..., 5] = 0.0
    k[at], v[at] = 0.0, 0.0
    k[at, :, 5] = octaves * np.log(2) / (4.0 * SCALE)
    kr, vr = (oi.quantise(oi.bf16(x.numpy())) for x in (k, v))
    q = q.to(torch.bfloat16)
    lse = torch.empty((B * nq, 32), device="cuda")
    cache, table = _cache(kr, vr)
    out, _ = ops.paged_prefill_attention_int4(q.cuda(), cache, table.repeat(B, 1), np.arange(B + 1) * nq, [n - nq] * B, [n] * B, True,
                                              lse=lse)
    vis = np.arange(n)[None] <= n - nq + np.arange(nq)[:, None]
    for b in (0, B - 1):
        mine = slice(b * nq, (b + 1) * nq)
        want, want_lse, tol, ltol = oi.attend(q[mine].double().numpy(), kr, vr, vis, SCALE, wide=True)
        # the floor of a weight, 2^-36 of the largest, on every row's value, and through the sum's own error
        tol = tol + 2.0 ** -36 * n * (np.abs(oi.values(vr)).max() + np.abs(want))
        err = np.abs(out[mine].double().cpu().numpy() - want)
        assert (err <= tol).all(), (err.max(), tol.min(), np.abs(want).max())
        assert (np.abs(lse[mine].double().cpu().numpy() - want_lse) <= ltol + 2.0 ** -36 * n).all()
