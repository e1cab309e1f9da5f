"""Single-token attention over a cache in 4 bits where no split rounds anything: what the output's own rounding allows."""
import numpy as np
import pytest
import torch

from oracle import int4 as oi

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


@pytest.mark.parametrize("shift", [0.0, 3.0])
@pytest.mark.parametrize("split_pages", [64, 0])
def test_weights_keep_their_bits(split_pages, shift):
    """Sequences that one workgroup takes whole: an output is as exact as its rounding to bf16 and fp32 sums leave it, and the same
    rows as a chunk of one query (fp16 values and weights, the same rounding) give no more exact ones."""
    from abridgekv_amd import ops
    lens = [2, 3, 5, 9, 17, 32, 64, 100, 333, 1000]
    gen = torch.Generator().manual_seed(9)
    B, W = len(lens), 63
    q = torch.randn((B, 32, 128), generator=gen).to(torch.bfloat16)
    cache = np.zeros((B * W, 2, 16, 640), np.uint8)
    table = np.arange(B * W, dtype=np.int32).reshape(B, W)
    rows = []
    for b, n in enumerate(lens):
        k, v = (torch.randn((n, 8, 128), generator=gen) for _ in range(2))
        rows.append([oi.quantise(oi.bf16(x.numpy())) for x in (k, v + shift)])
        at = np.arange(n)
        for half in (0, 1):
            cache[table[b, at // 16], half, at % 16] = rows[b][half]
    cache, dev = torch.from_numpy(cache).cuda(), torch.from_numpy(table).cuda()
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    if split_pages:
        out, _ = ops.decode_attention_int4(q.cuda(), cache, dev, sl, split_pages=split_pages)
    else:                                                    # shares: one at a time, of at most two pages, is one share
        out = torch.cat([ops.decode_attention_int4(q[b: b + 1].cuda(), cache, dev[b: b + 1], sl[b: b + 1], split_pages=0,
                                                   max_pages=2)[0] for b in range(6)])
    one, _ = ops.paged_prefill_attention_int4(q.cuda(), cache, dev, np.arange(B + 1), [n - 1 for n in lens], lens, True)
    mine = theirs = 0.0
    for b in range(len(out)):
        want, _, tol, _ = oi.attend(q[b: b + 1].double().numpy(), *rows[b], np.ones((1, lens[b]), bool), SCALE, whole=True)
        err, other = (np.abs(x[b: b + 1].double().cpu().numpy() - want) for x in (out, one))
        assert (err <= tol).all(), (lens[b], (err - tol).max())
        mine, theirs = mine + (err ** 2).sum() / (want ** 2).sum(), theirs + (other ** 2).sum() / (want ** 2).sum()
    assert mine <= 1.1 * theirs
