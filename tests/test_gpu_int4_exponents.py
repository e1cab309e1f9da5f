"""Multi-query attention over a cache in 4 bits: queries and keys whose powers of two are far apart, against the float64 oracle."""
import numpy as np
import pytest
import torch

from oracle import int4 as oi

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


@pytest.mark.parametrize("of_q,of_k", [(-95, lambda p: 95), (-108, lambda p: 110), (100, lambda p: -100),
                                       (-95, lambda p: (95, 40, 97)[p % 3])])
def test_tiny_queries_and_huge_keys(of_q, of_k):
    from abridgekv_amd import ops
    n, nq = 300, 40
    gen = torch.Generator().manual_seed(4)
    k, v = (torch.randn((n, 8, 128), generator=gen) for _ in range(2))
    k *= torch.tensor([2.0 ** of_k(i // 16) for i in range(n)])[:, None, None]
    q = (torch.randn((nq, 32, 128), generator=gen) * 2.0 ** of_q).to(torch.bfloat16)
    kr, vr = (oi.quantise(oi.bf16(x.numpy())) for x in (k, v))
    pages = -(-n // 16)
    cache = np.zeros((pages, 2, 16, 640), np.uint8)
    at = np.arange(n)
    cache[at // 16, 0, at % 16], cache[at // 16, 1, at % 16] = kr, vr
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    lse = torch.empty((nq, 32), device="cuda")
    out, _ = ops.paged_prefill_attention_int4(q.cuda(), torch.from_numpy(cache).cuda(), table, [0, nq], [n - nq], [n], True, lse=lse)
    vis = np.arange(n)[None] <= n - nq + np.arange(nq)[:, None]
    want, want_lse, tol, ltol = oi.attend(q.double().numpy(), kr, vr, vis, SCALE, wide=True)
    assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()
    assert (np.abs(lse.double().cpu().numpy() - want_lse) <= ltol).all()
