"""The custom ops of a windowed training step: the forward that leaves the outputs' low part and the backward that takes it."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from abridgekv_amd import ops, torch_ops

SCALE = 128 ** -0.5


def test_registered_with_its_mutations():
    assert torch_ops.TRAINING_OPS == ("window_attn_low",)
    schema = torch.ops.abridgekv.window_attn_low.default._schema
    assert {a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write} == {"out", "lse", "out_low"}
    assert len(schema.returns) == 0
    low = torch.ops.abridgekv.window_attn_bwd.default._schema.arguments[-1]
    assert low.name == "out_low" and low.has_default_value() and low.default_value is None


def test_fake_tracing_keeps_a_step_as_two_nodes():
    def step(q, k, lens, out, lse, low):
        torch.ops.abridgekv.window_attn_low(q, k, k, 16, 2, lens, SCALE, out, lse, low)
        return torch.ops.abridgekv.window_attn_bwd(q, k, k, out, lse, out, 16, 2, lens, SCALE, low)

    with FakeTensorMode():
        q, out = (torch.empty((2, 24, 32, 128), device="cuda", dtype=torch.bfloat16) for _ in range(2))
        gm = make_fx(step, tracing_mode="fake")(q, torch.empty((2, 24, 8, 128), device="cuda", dtype=torch.bfloat16),
                                                torch.empty(2, device="cuda", dtype=torch.int32), out,
                                                torch.empty((2, 32, 24), device="cuda"),
                                                torch.empty((2, 24, 32, 128), device="cuda", dtype=torch.float8_e5m2))
        with pytest.raises(ValueError, match="out_low"):
            torch.ops.abridgekv.window_attn_low(q, q[:, :, :8], q[:, :, :8], 16, 2, None, SCALE, out, out, out[:1])
    names = [str(n.target) for n in gm.graph.nodes if n.op == "call_function"]
    assert sum(n.startswith("abridgekv.") for n in names) == 2


def _qkvg(seed, S=150):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn((2, S, h, 128), generator=gen).to(torch.bfloat16).cuda() for h in (32, 8, 8, 32)]


@pytest.mark.gpu
def test_steps_match_direct_calls_and_autograd():
    import types

    from abridgekv_amd.compress_forward import WindowMask, masked_attention_forward
    T = torch.ops.abridgekv
    q, k, v, g = _qkvg(7)
    sl = torch.tensor([150, 61], dtype=torch.int32, device="cuda")

    def buffers():
        return (torch.empty_like(q), torch.empty((2, 32, 150), device="cuda"),
                torch.empty(q.shape, dtype=torch.float8_e5m2, device="cuda"))

    out, lse, low = buffers()
    T.window_attn_low(q, k, v, 50, 3, sl, SCALE, out, lse, low)
    grads = T.window_attn_bwd(q, k, v, out, lse, g, 50, 3, sl, SCALE, low)
    want, wlse, wlow = buffers()
    ops.window_attention(q, k, v, 50, 3, seq_lens=sl, scale=SCALE, out=want, lse=wlse, out_low=wlow)
    direct = ops.window_attention_backward(q, k, v, want, wlse, g, 50, 3, seq_lens=sl, scale=SCALE, out_low=wlow)
    assert torch.equal(out, want) and torch.equal(lse, wlse)
    assert torch.equal(low.view(torch.uint8), wlow.view(torch.uint8))
    assert all(torch.equal(a, b) for a, b in zip(grads, direct))
    leaves = [t.transpose(1, 2).requires_grad_(True) for t in (q, k, v)]
    out, _ = masked_attention_forward(types.SimpleNamespace(layer_idx=0), *leaves, WindowMask(50, 3, sl))
    auto = torch.autograd.grad(out, leaves, g)
    assert all(torch.equal(a, b.transpose(1, 2)) for a, b in zip(grads, auto))
    # without it: other bits of dq and dk, the same dv
    plain = T.window_attn_bwd(q, k, v, want, wlse, g, 50, 3, sl, SCALE)
    assert not torch.equal(plain[0], grads[0]) and not torch.equal(plain[1], grads[1]) and torch.equal(plain[2], grads[2])
