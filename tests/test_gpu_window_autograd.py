"""Sliding-window attention under ``create_graph``: first gradients are those without it, a second derivative is refused."""
import types

import pytest
import torch

pytestmark = pytest.mark.gpu


def _call(seed, grad=(True, True, True)):
    from abridgekv_amd.compress_forward import WindowMask, masked_attention_forward
    gen = torch.Generator().manual_seed(seed)
    qkv = [torch.randn((2, h, 90, 128), generator=gen).to(torch.bfloat16).cuda().requires_grad_(r)
           for h, r in zip((32, 8, 8), grad)]
    dout = torch.randn((2, 90, 32, 128), generator=gen).to(torch.bfloat16).cuda()
    out, _ = masked_attention_forward(types.SimpleNamespace(layer_idx=0), *qkv, WindowMask(40, 3))
    return qkv, out, dout


def test_first_gradients_with_create_graph():
    qkv, out, dout = _call(1)
    want = torch.autograd.grad(out, qkv, dout)
    qkv, out, dout = _call(1)
    got = torch.autograd.grad(out, qkv, dout, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # a loss that takes no second derivative of the attention beside others that do
    qkv, out, dout = _call(1)
    w = torch.ones((), device="cuda", requires_grad=True)
    (gw,) = torch.autograd.grad((out.float() * dout.float()).sum() * w ** 3, w, create_graph=True)
    (ggw,) = torch.autograd.grad(gw, w)
    assert torch.allclose(ggw, 2 * gw, rtol=1e-4)


@pytest.mark.parametrize("grad", [(True, True, True), (True, False, False), (False, True, False), (False, False, True)])
@pytest.mark.parametrize("through_dout", [False, True])
def test_second_derivatives_are_refused(grad, through_dout):
    """Whichever input they go through, and that of the gradient handed in."""
    qkv, out, dout = _call(2, grad)
    dout.requires_grad_(through_dout)
    leaves = [t for t in qkv if t.requires_grad]
    first = torch.autograd.grad(out, leaves, dout, create_graph=True)
    loss = sum((g.float() ** 2).sum() for g in first)
    for leaf in leaves + [dout] * through_dout:
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(loss, leaf, retain_graph=True)
