"""Log probabilities with and without the entropy, which are kernels of their own: the same bits, NaNs among them."""
import pytest
import torch

from test_gpu_logprobs import SIZES, _logits

pytestmark = pytest.mark.gpu


def _same(a, b):
    assert a.dtype == b.dtype and a.shape == b.shape
    assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(nan=7.0), b.nan_to_num(nan=7.0))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,V,n", SIZES)
def test_without_entropy(T, V, n, dt):
    """Banned tokens, rows without a target, and a NaN or an infinity in every fifth row."""
    from abridgekv_amd import ops
    x, t = _logits(T, V, dt, T + V, banned=V // 10)
    t[::4] = -100
    x[4::5, V // 2] = float("nan")
    x[3::5, V // 3] = float("inf")
    x, t = x.cuda(), t.cuda()
    got = ops.token_logprobs(x, t, 0.7, top=n)
    again = ops.token_logprobs(x, t, 0.7, top=n, entropy=False)
    assert got.entropy is not None and again.entropy is None and got.stats is None and again.stats is None
    _same(again.logprob, got.logprob)
    _same(again.top_logprobs, got.top_logprobs)
    assert torch.equal(again.top_ids, got.top_ids)
    if T > 4:
        assert got.logprob[1::5].isnan().sum() == 0 and got.entropy[4::5].isnan().all()
