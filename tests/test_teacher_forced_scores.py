"""Chunk sizes of the training wrapper's ``token_logprobs``, on the CPU with the kernel's call in plain torch."""
import types

import pytest
import torch

from abridgekv_amd import ops
from abridgekv_amd.compress_forward import CompressLM


def _plain(logits, targets, temperature=1.0, top=0):
    ls = torch.log_softmax(logits.float() / temperature, -1)
    best = torch.sort(ls, dim=-1, descending=True, stable=True)
    return ops.TokenLogprobs(ls.gather(1, targets[:, None])[:, 0], -(ls.exp() * ls).sum(-1), best.indices[:, :top], best.values[:, :top], None)


@pytest.mark.parametrize("rows", [7, 0])
@pytest.mark.parametrize("chunk", [4096, 7, 3, 0, -1])
def test_chunks(rows, chunk, monkeypatch):
    """``chunk`` <= 0 takes all rows at once, as in the losses; no rows at all give empty results."""
    monkeypatch.setattr(ops, "token_logprobs", _plain)
    gen = torch.Generator().manual_seed(1)
    hid = torch.randn((2, 9, 16), generator=gen)
    head = torch.nn.Linear(16, 30)
    lm = types.SimpleNamespace(hidden_states=lambda ids, prompt_len: hid, loss_pos=torch.arange(9) < rows,
                               predict_flat=torch.arange(rows), model=types.SimpleNamespace(
                                   config=types.SimpleNamespace(hidden_size=16), lm_head=head))
    ids = torch.randint(0, 30, (2, 1, 12), generator=gen)
    got = CompressLM.token_logprobs(lm, ids, temperature=0.8, top=3, chunk=chunk)
    want = _plain(head(hid[:, :rows].reshape(-1, 16)).detach(), ids[:, 0, 1: 1 + rows].reshape(-1), 0.8, 3)
    for a, b in zip(got[:4], want[:4]):
        assert a.shape == b.shape and torch.allclose(a.double(), b.double(), atol=1e-5)
    assert got.stats is None
