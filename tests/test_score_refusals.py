"""The generator's ``score`` refuses what it cannot answer before it feeds anything, on the CPU."""
import types

import pytest
import torch

from abridgekv_amd.gen_compress import CompressGen


def _gen(fed):
    def feed_content(ids):
        fed.append(ids)
        raise RuntimeError("fed")

    return types.SimpleNamespace(C=64, f=0, b=0, device="cpu", feed_content=feed_content, compress=lambda: fed.append(None),
                                 lm_head=torch.nn.Linear(4, 100), inner=types.SimpleNamespace(embed_tokens=torch.nn.Embedding(100, 4)))


@pytest.mark.parametrize("answer,kw,match", [
    ([5, 100], {}, "token"), ([5, -1], {}, "token"), ([100, 5], {}, "token"), ([], {}, "answer"),
    ([5, 6], {"top": 33}, "top"), ([5, 6], {"top": -1}, "top"), ([5, 6], {"temperature": 0.0}, "temperature"),
    ([5, 6], {"temperature": 1e30}, "temperature"), ([5, 6], {"temperature": float("nan")}, "temperature")])
def test_score(answer, kw, match):
    fed = []
    with pytest.raises(ValueError, match=match):
        CompressGen.score(_gen(fed), [1, 2, 3], answer, **kw)
    assert not fed


def test_score_of_a_bad_prompt_and_a_good_call():
    fed = []
    for prompt in ([1, 100], [-3, 1], []):
        with pytest.raises(ValueError):
            CompressGen.score(_gen(fed), prompt, [5, 6])
    assert not fed
    with pytest.raises(RuntimeError, match="fed"):
        CompressGen.score(_gen(fed), [0, 99], [99, 0], top=32)
    assert fed == [[0, 99, 99]]
