"""Temperatures that the log probabilities refuse, on the CPU."""
import pytest
import torch

from abridgekv_amd import fused, ops
from abridgekv_amd._lib import lib


def test_temperatures_out_of_range():
    """A banned logit counts as -1e25, so at a temperature near that it would weigh something; the reciprocal of a tiny one is no
    float. Both are refused, here and at the C entries; what lies between gets as far as the device check."""
    x, t = torch.zeros((3, 50)), torch.zeros(3, dtype=torch.int64)
    st, g = torch.zeros((3, 3)), torch.zeros(3)
    calls = (lambda T: ops.token_logprobs(x, t, T), lambda T: fused.token_logprobs(x, t, T),
             lambda T: ops.token_logprobs_backward(x, t, st, g, None, T))
    for call in calls:
        for bad in (1e-45, 1e-39, 9e-31, 1.1e20, 1e26, 3e38):
            with pytest.raises(ValueError, match="temperature"):
                call(bad)
        for good in (1e-30, 0.01, 100.0, 1e20):
            with pytest.raises(ValueError, match="current GPU"):
                call(good)
    L = lib()
    p = torch.zeros(1 << 16, dtype=torch.uint8)
    a = p.data_ptr() + (-p.data_ptr()) % 16
    for bad in (1e-39, 9e-31, 1.1e20, 1e26, float("inf"), float("nan")):
        assert L.abkv_token_logprobs(0, a, 50, 2, 50, a, bad, 0, a, a, a, a, a, a, 1 << 20, None) != 0
        assert L.abkv_token_logprobs_bwd(0, a, 50, 2, 50, a, bad, a, a, a, a, 50, None) != 0
