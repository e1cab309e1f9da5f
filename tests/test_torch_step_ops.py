"""The custom-op registrations of the step operators, without a GPU: mutation schemas, and one graph node each under fake
tracing."""
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from abridgekv_amd import torch_ops

MUTATES = {
    "kv_append_int4": {"kv_cache"},
    "decode_attn_int4": {"out", "lse", "workspace"},
    "qk_norm_rope_append": {"kv_cache", "out"},
    "qk_norm_rope": set(),
    "qk_norm_rope_bwd": set(),
    "token_logprobs": set(),
    "token_logprobs_bwd": set(),
}


def test_every_op_is_registered_with_its_mutations():
    assert set(torch_ops.STEP_OPS) == set(MUTATES)
    for name, muts in MUTATES.items():
        schema = getattr(torch.ops.abridgekv, name).default._schema
        assert {a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write} == muts, name
        assert (len(schema.returns) == 0) == bool(muts), name


def test_fake_tracing_keeps_each_op_as_one_node():
    T = torch.ops.abridgekv

    def caller(q, k, out, cache, table, lens, slots, cs, w, ws, tq, tk, cos, logits, targets):
        T.qk_norm_rope_append(q, k, k, slots, cs, slots, cache, w, w, 1e-6, 0, 0, 5, 0, out)
        T.kv_append_int4(k, k, slots, cache)
        T.decode_attn_int4(out, cache, table, lens, 0.088, 8, 4, q, None, ws)
        a, b = T.qk_norm_rope(tq, tk, cos, cos, w, w, 1e-6)
        c, d, e, f = T.qk_norm_rope_bwd(tq, tk, a, b, cos, cos, w, w, 1e-6)
        lp, ent, ids, tops, stats = T.token_logprobs(logits, targets, 1.0, 3)
        g = T.token_logprobs_bwd(logits, targets, stats, lp, ent, 1.0)
        return c.sum() + d.sum() + e.sum() + f.sum() + g.sum() + tops.sum() + ids.sum()

    with FakeTensorMode():
        bf, dev = torch.bfloat16, "cuda"
        args = (torch.empty(2, 32, 128, device=dev, dtype=bf), torch.empty(2, 8, 128, device=dev, dtype=bf),
                torch.empty(2, 32, 128, device=dev, dtype=bf), torch.empty(40, 2, 16, 640, device=dev, dtype=torch.uint8),
                torch.empty(2, 8, device=dev, dtype=torch.int32), torch.empty(2, device=dev, dtype=torch.int32),
                torch.empty(2, device=dev, dtype=torch.int64), torch.empty(9, 128, device=dev),
                torch.empty(128, device=dev, dtype=bf), torch.empty(1 << 16, device=dev, dtype=torch.uint8),
                torch.empty(2, 7, 32, 128, device=dev, dtype=bf), torch.empty(2, 7, 8, 128, device=dev, dtype=bf),
                torch.empty(1, 7, 128, device=dev, dtype=bf), torch.empty(4, 100, device=dev, dtype=bf),
                torch.empty(4, device=dev, dtype=torch.int64))
        graph = make_fx(caller, tracing_mode="fake")(*args)
    names = [str(n.target) for n in graph.graph.nodes if n.op == "call_function"]
    for op in torch_ops.STEP_OPS:
        assert sum(n == f"abridgekv.{op}.default" for n in names) == 1, op
