"""Fused operators with gradients, and a model's attention layers on them.

``qk_norm_rope``: RMS norms of queries and keys for each head and their rotation; ``token_logprobs``: log probabilities of given
tokens and the distribution's entropy. Forward and backward are one kernel each (and a small one for the norms' weights). As with
any autograd function, a backward pass is captured into a graph only when no eager graph of the same leaves is alive.
"""
from __future__ import annotations

import torch

from . import ops


class _FirstDerivative(torch.autograd.Function):
    """Gradients that a kernel made, tied to what they were made from: a second derivative through them is refused."""

    @staticmethod
    def forward(ctx, name, count, *tensors):
        ctx.name = name
        return tuple(t.view_as(t) for t in tensors[:count])

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"{ctx.name} has no second derivative")


def _gradient_rows(g: torch.Tensor) -> torch.Tensor:
    """An upstream gradient as the kernels read it (autograd hands over expanded or transposed ones)."""
    st, e = g.stride(), g.element_size()
    dense = st[3] == 1 and (st[0] | st[1] | st[2]) * e % 16 == 0 and st[1] < 1 << 24 and g.data_ptr() % 16 == 0
    return g if dense else g.contiguous()


class _QKNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, cos, sin, q_weight, k_weight, eps):
        ctx.save_for_backward(q, k, cos, sin, q_weight, k_weight)
        ctx.eps = eps
        return ops.qk_norm_rope(q, k, cos, sin, q_weight, k_weight, eps)

    @staticmethod
    def backward(ctx, dq_out, dk_out):
        q, k, cos, sin, q_weight, k_weight = ctx.saved_tensors
        grads = ops.qk_norm_rope_backward(q, k, _gradient_rows(dq_out), _gradient_rows(dk_out), cos, sin, q_weight, k_weight,
                                          ctx.eps)
        if torch.is_grad_enabled():                          # (create_graph)
            grads = _FirstDerivative.apply("qk_norm_rope", 4, *grads, q, k, q_weight, k_weight, dq_out, dk_out)
        dq, dk, dwq, dwk = grads
        return dq, dk, None, None, dwq, dwk, None


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, q_weight: torch.Tensor,
                 k_weight: torch.Tensor, eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """:func:`ops.qk_norm_rope` with gradients of q, k and both weights (cos and sin take none; no second derivative)."""
    if cos.requires_grad or sin.requires_grad:
        raise NotImplementedError("the angles take no gradient")
    return _QKNormRope.apply(q, k, cos, sin, q_weight, k_weight, float(eps))


def head_norms(attn):
    """(q weight, k weight, eps) of an attention layer's per-head RMS norms, (None, None, 0.0) of a layer without any; norms of
    another kind are refused."""
    qn, kn = getattr(attn, "q_norm", None), getattr(attn, "k_norm", None)
    if qn is None and kn is None:
        return None, None, 0.0
    eps = [getattr(n, "variance_epsilon", None) for n in (qn, kn)]
    weights = [getattr(n, "weight", None) for n in (qn, kn)]
    if None in eps or eps[0] != eps[1] or any(w is None or w.shape != (ops.HEAD_DIM,) for w in weights):
        raise NotImplementedError("the fused norms take RMS norms of queries and keys over a head's 128 dims")
    return weights[0], weights[1], float(eps[0])


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, temperature):
        got = ops.token_logprobs(logits, targets, temperature, stats=True)
        ctx.save_for_backward(logits, targets, got.stats)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        return got.logprob, got.entropy

    @staticmethod
    def backward(ctx, dlogprob, dentropy):
        logits, targets, stats = ctx.saved_tensors
        if dlogprob is None and dentropy is None:
            return None, None, None
        g, h = (t if t is None else t.contiguous() for t in (dlogprob, dentropy))
        grad = ops.token_logprobs_backward(logits, targets, stats, g, h, ctx.temperature)
        if torch.is_grad_enabled():                          # (create_graph)
            sources = [t for t in (logits, dlogprob, dentropy) if t is not None]
            (grad,) = _FirstDerivative.apply("token_logprobs", 1, grad, *sources)
        return grad, None, None


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, temperature: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """(log probability, entropy) [T] fp32 of :func:`ops.token_logprobs` with the gradient of the logits [T, V] (no second
    derivative). Rows whose target lies outside [0, V) have log probability 0 and no gradient from it."""
    return _TokenLogprobs.apply(logits, targets, float(temperature))
