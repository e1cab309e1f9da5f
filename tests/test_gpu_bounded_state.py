"""The state of a cache bounded by weight: layers of their own, sequences inside their budget, and scored steps of one split."""
import numpy as np
import pytest
import torch

from oracle import evict as oe
from oracle import window as ow

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


def _state(seed, lens, layers, spare=3, garbage=float("nan")):
    """Layer caches of different rows under one table, scores and positions as a run before would have left them."""
    rng = np.random.default_rng(seed)
    gen = torch.Generator().manual_seed(seed)
    need = [-(-n // 16) for n in lens]
    W, pool = max(need) + 1, sum(need) + spare
    pages = rng.permutation(pool)[: sum(need)]
    table = np.zeros((len(lens), W), np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = pages[at: at + n]
        at += n
    caches = []
    for _ in range(layers):
        c = torch.full((pool, 2, 16, 8, 128), garbage, dtype=torch.bfloat16)
        for b, n in enumerate(lens):
            s = np.arange(n)
            c[torch.from_numpy(table[b, s // 16].astype(np.int64)), :, torch.from_numpy(s % 16)] = torch.randn(
                (n, 2, 8, 128), generator=gen).to(torch.bfloat16)
        caches.append(c.cuda())
    scores = torch.rand((layers, len(lens), 8, W * 16), generator=gen)
    positions = torch.full((layers, len(lens), 8, W * 16), -1, dtype=torch.int32)
    return caches, torch.from_numpy(table).cuda(), scores.cuda(), positions.cuda()


def _rows(cache, table, b, n):
    s = torch.arange(n, device="cuda")
    return cache[table[b, s // 16].long(), :, s % 16]


@pytest.mark.parametrize("budget", [100, 129])
def test_sequences_inside_their_budget_are_left_alone(budget):
    """Beside ones that are not: rows, scores and positions keep their bits, and so do rows past every sequence."""
    from abridgekv_amd import ops
    lens = [budget, 300, budget - 1, 1, 0, budget + 1]
    caches, table, scores, positions = _state(budget, lens, 2)
    before = [c.clone() for c in caches], scores.clone(), positions.clone()
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    new = ops.kv_evict(caches, table, sl, scores, positions, sl.clone(), budget, 4, 20)
    assert new.tolist() == [min(n, budget) for n in lens]
    for b, n in enumerate(lens):
        if n <= budget:
            assert torch.equal(scores[:, b], before[1][:, b]) and torch.equal(positions[:, b], before[2][:, b])
            for c, old in zip(caches, before[0]):
                assert torch.equal(_rows(c, table, b, n), _rows(old, table, b, n))
        else:
            assert (scores[:, b, :, n:] == before[1][:, b, :, n:]).all() and (positions[:, b, :, n:] == -1).all()
            assert (scores[:, b, :, budget:n] == 0).all() and (positions[:, b, :, budget:n] == -1).all()
            assert (positions[:, b, :, :budget] >= 0).all()
    for c, old in zip(caches, before[0]):
        lost = torch.isnan(old)
        assert torch.equal(torch.isnan(c), lost)                          # rows of no sequence


def test_each_layer_keeps_its_own_rows():
    """Three layers with scores of their own, twice with appended rows between: every kept row is the token's that its position
    names, in the layer and head it belongs to, and the kept tokens are the oracle's."""
    from abridgekv_amd import ops
    layers, lens, budget, sinks, recent = 3, [150, 90], 64, 3, 10
    caches, table, scores, positions = _state(5, lens, layers)
    tokens = list(lens)
    kv = [[{t: row for t, row in enumerate(_rows(c, table, b, n).cpu())} for b, n in enumerate(lens)] for c in caches]
    have = [[[list(range(n)) for _ in range(8)] for n in lens] for _ in caches]
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    gen = torch.Generator().manual_seed(9)
    for _ in range(2):
        old = scores.cpu()
        sl = ops.kv_evict(caches, table, sl, scores, positions, torch.tensor(tokens, dtype=torch.int32, device="cuda"), budget,
                          sinks, recent)
        for l in range(layers):
            for b in range(2):
                now = _rows(caches[l], table, b, budget).cpu()
                for h in range(8):
                    toks = have[l][b][h]
                    n = len(toks)
                    want = oe.evict(old[l, b, h, :n].double().numpy().tolist(), toks, tokens[b], budget, sinks, recent)
                    got = positions[l, b, h, :budget].tolist()
                    assert set(got) == {int(x) for x in want[2][:budget]}, (l, b, h)
                    at = {t: i for i, t in enumerate(toks)}
                    assert scores[l, b, h, :budget].tolist() == [float(old[l, b, h, at[t]]) for t in got]
                    assert all(torch.equal(now[i, :, h], kv[l][b][t][:, h]) for i, t in enumerate(got)), (l, b, h)
                    have[l][b][h] = got
        for _ in range(20):                                  # rows appended behind, the same tokens in every layer
            n = sl.tolist()
            for l, c in enumerate(caches):
                for b in range(2):
                    row = torch.randn((2, 8, 128), generator=gen).to(torch.bfloat16)
                    c[int(table[b, n[b] // 16]), :, n[b] % 16] = row.cuda()
                    kv[l][b][tokens[b]] = row
                    for h in range(8):
                        have[l][b][h].append(tokens[b])
                    scores[l, b, :, n[b]] = torch.rand(8, generator=gen).cuda()
            tokens = [t + 1 for t in tokens]
            sl = sl + 1


def test_scored_step_of_one_split():
    """A split of every page (eight waves share it, its scores go through memory): sequences too long for a workgroup of their own."""
    from abridgekv_amd import ops
    lens = [1000, 500, 7, 0]
    caches, table, scores, _ = _state(11, lens, 1)
    q = torch.randn((4, 32, 128), generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    start = scores[0].clone()
    lse = torch.empty((4, 32), device="cuda")
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out, _ = ops.decode_attention_scored(q.cuda(), caches[0], table, sl, scores[0], lse=lse, split_pages=64)
    for b, n in enumerate(lens):
        added = (scores[0, b].double() - start[b].double()).cpu().numpy()
        assert not added[:, n:].any()
        if n == 0:
            assert not out[b].any()
            continue
        k, v = _rows(caches[0], table, b, n).double().cpu().numpy().transpose(1, 0, 2, 3)
        vis = np.ones((1, n), bool)
        want, want_lse, _, tol = ow.attend(q[b: b + 1].double().numpy(), k, v, vis, SCALE, True)
        # (the split's partial is fp16: 2^-11 of its largest |out|)
        assert (np.abs(out[b].double().cpu().numpy() - want[0]) <= tol[0] + 2.0 ** -11 * np.abs(v).max()).all()
        assert np.abs(lse[b].double().cpu().numpy() - want_lse[0]).max() <= 1e-4
        w = oe.weights(q[b: b + 1].double().numpy(), k, v, [n - 1], SCALE)
        # weights in fp32 (128-term scores of |q . k| up to about 50: 4e-5), added to scores below 1 (a rounding of 2^-24 x 5)
        assert np.abs(added[:, :n] - w).max() <= 4e-5 + 5 * 2.0 ** -24
