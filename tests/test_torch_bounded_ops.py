"""The custom-op registrations of the window, score and eviction operators, without a GPU: mutation schemas, and one graph
node each under fake tracing."""
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from abridgekv_amd import torch_ops

MUTATES = {
    "decode_attn_window": {"out", "lse", "workspace"},
    "decode_attn_scored": {"scores", "out", "lse", "workspace"},
    "kv_evict": {"layer_caches", "scores", "positions", "out_lens", "workspace"},
    "window_attn": {"out", "lse"},
    "window_attn_bwd": set(),
}


def test_every_op_is_registered_with_its_mutations():
    assert set(torch_ops.BOUNDED_OPS) == set(MUTATES)
    for name, muts in MUTATES.items():
        schema = getattr(torch.ops.abridgekv, name).default._schema
        got = {a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write}
        assert got == muts, (name, got)
        assert (len(schema.returns) == 0) == (name != "window_attn_bwd"), name


def test_fake_tracing_keeps_each_op_as_one_node():
    def caller(q, cache, table, lens, out, lse, ws, scores, positions, tokens, new_lens, pq, pk, pout, plse):
        torch.ops.abridgekv.decode_attn_window(q, cache, table, lens, 64, 4, 0.088, 8, 4, out, lse, ws)
        torch.ops.abridgekv.decode_attn_scored(q, cache, table, lens, scores[0], 0.088, 8, 4, out, lse, ws)
        torch.ops.abridgekv.kv_evict([cache], table, lens, scores, positions, tokens, 64, 4, 16, 8, new_lens, None)
        torch.ops.abridgekv.window_attn(pq, pk, pk, 16, 2, lens, 0.088, pout, plse)
        dq, dk, dv = torch.ops.abridgekv.window_attn_bwd(pq, pk, pk, pout, plse, pout, 16, 2, lens, 0.088)
        return out.sum() + dq.float().sum() + dk.float().sum() + dv.float().sum()

    with FakeTensorMode():
        d, bf, i32 = "cuda", torch.bfloat16, torch.int32
        args = (torch.empty(2, 32, 128, device=d, dtype=bf), torch.empty(40, 2, 16, 8, 128, device=d, dtype=bf),
                torch.empty(2, 8, device=d, dtype=i32), torch.empty(2, device=d, dtype=i32),
                torch.empty(2, 32, 128, device=d, dtype=bf), torch.empty(2, 32, device=d),
                torch.empty(1 << 16, device=d, dtype=torch.uint8), torch.empty(1, 2, 8, 128, device=d),
                torch.empty(1, 2, 8, 128, device=d, dtype=i32), torch.empty(2, device=d, dtype=i32),
                torch.empty(2, device=d, dtype=i32), torch.empty(2, 24, 32, 128, device=d, dtype=bf),
                torch.empty(2, 24, 8, 128, device=d, dtype=bf), torch.empty(2, 24, 32, 128, device=d, dtype=bf),
                torch.empty(2, 32, 24, device=d))
        gm = make_fx(caller, tracing_mode="fake")(*args)
    targets = [str(n.target) for n in gm.graph.nodes if n.op == "call_function"]
    for name in torch_ops.BOUNDED_OPS:
        assert sum(t.startswith(f"abridgekv.{name}.") for t in targets) == 1, (name, targets)
