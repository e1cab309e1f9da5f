"""Log probabilities at the ends of the temperatures that they take."""
import pytest
import torch

from test_gpu_logprobs import _logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("temperature", [1e-30, 1e20])
def test_the_widest_temperatures(temperature):
    """At 1e20 every token that is not banned is as likely as any other, and a banned one never; at 1e-30 the largest is alone."""
    from abridgekv_amd import ops
    x, t = _logits(3, 1000, torch.float32, 5)
    x[:, ::2] = -float("inf")
    t[:] = x.argmax(1)
    got = ops.token_logprobs(x.cuda(), t.cuda(), temperature, top=2)
    want = 0.0 if temperature < 1 else -torch.tensor(500.0).log()
    assert torch.allclose(got.logprob.cpu(), torch.full((3,), float(want)), rtol=1e-5, atol=0)
    assert torch.allclose(got.entropy.cpu(), torch.full((3,), -float(want)), rtol=1e-5, atol=0)
    grad = ops.token_logprobs_backward(x.cuda(), t.cuda(), ops.token_logprobs(x.cuda(), t.cuda(), temperature, stats=True).stats,
                                       torch.ones(3, device="cuda"), torch.ones(3, device="cuda"), temperature)
    assert not grad[:, ::2].any() and grad.isfinite().all()
