"""Multi-query attention over a cache in 4 bits with key rows that read as NaN: out and lse, where they are seen and elsewhere."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,nq", [(300, 40), (4061, 61)], ids=["one part", "many parts"])
def test_keys_that_are_not_finite(n, nq):
    """A NaN group of keys makes out and lse of its KV head NaN, as single tokens over the same rows have it; a row that sees
    nothing keeps lse -inf, and every other row its bits."""
    from abridgekv_amd import ops
    gen = torch.Generator().manual_seed(n)
    k, v = (torch.randn((n, 8, 128), generator=gen).to(torch.bfloat16).cuda() for _ in range(2))
    q = torch.randn((nq + 3, 32, 128), generator=gen).to(torch.bfloat16).cuda()
    pages = -(-n // 16)
    cache = torch.zeros(ops.kv_cache_int4_shape(pages), dtype=torch.uint8, device="cuda")
    ops.kv_append_int4(k, v, torch.arange(n, device="cuda"), cache)
    table = torch.arange(pages, dtype=torch.int32, device="cuda").repeat(2, 1)
    args = (table, [0, nq, nq + 3], [n - nq, 0], [n, 0], True)
    lse, good_lse = (torch.empty((nq + 3, 32), device="cuda") for _ in range(2))
    good, _ = ops.paged_prefill_attention_int4(q, cache, *args, lse=good_lse)
    pairs = cache[1, 0, 3, 512 + 16 * 2 + 4: 512 + 16 * 2 + 6]                   # key row 19, head 2, group 1
    pairs.copy_(torch.tensor([0xC0, 0x7F], dtype=torch.uint8))
    out, _ = ops.paged_prefill_attention_int4(q, cache, *args, lse=lse)
    assert out[:nq, 8:12].isnan().all() and lse[:nq, 8:12].isnan().all()
    one_lse = torch.empty((1, 32), device="cuda")
    ops.decode_attention_int4(q[nq - 1: nq], cache, table[:1], torch.tensor([n], dtype=torch.int32, device="cuda"), lse=one_lse)
    assert one_lse[0, 8:12].isnan().all() and not one_lse[0, :8].isnan().any()
    rest = torch.ones_like(lse, dtype=torch.bool)
    rest[:nq, 8:12] = False
    assert torch.equal(out[rest], good[rest]) and torch.equal(lse[rest], good_lse[rest])
    assert not out[nq:].any() and (lse[nq:] == -float("inf")).all()
