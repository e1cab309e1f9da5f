"""The windowed baseline of models whose layers have attention windows of their own."""
import copy

import pytest
import torch


def _model(layer_types):
    transformers = pytest.importorskip("transformers")
    torch.manual_seed(3)
    own = dict(use_sliding_window=True, sliding_window=24) if "sliding_attention" in layer_types else {}
    cfg = transformers.Qwen3Config(vocab_size=257, hidden_size=256, intermediate_size=512, num_hidden_layers=2,
                                   num_attention_heads=32, num_key_value_heads=8, head_dim=128, max_position_embeddings=4096,
                                   rope_parameters={"rope_theta": 1e6, "rope_type": "default"}, layer_types=layer_types, **own)
    cfg._attn_implementation = "eager"
    return transformers.Qwen3ForCausalLM(cfg).to(torch.bfloat16).eval()


MIXED, SLIDING = ["full_attention", "sliding_attention"], ["sliding_attention"] * 2


@pytest.mark.parametrize("layer_types", [MIXED, SLIDING])
def test_windows_of_their_own_are_refused(layer_types):
    from abridgekv_amd.compress_forward import CompressLM
    clm = CompressLM(_model(layer_types), 48, 1, 16, code_positions="appended")
    ids = torch.zeros((1, 1, 48), dtype=torch.int64)
    with pytest.raises(NotImplementedError, match="sliding_attention"):
        clm(ids, baseline=True, window=20, sinks=2)
    with pytest.raises(NotImplementedError, match="full-attention layers"):
        clm.baseline_loss(ids, window=20)


@pytest.mark.gpu
@pytest.mark.parametrize("layer_types", [MIXED, SLIDING])
def test_their_baseline_without_a_window_runs(layer_types):
    """Layers with windows of their own run them, so the loss is another than full attention's."""
    from abridgekv_amd.compress_forward import CompressLM
    base = _model(layer_types)
    ids = torch.randint(0, 257, (2, 1, 192), generator=torch.Generator().manual_seed(1)).cuda()
    with torch.no_grad():
        got = CompressLM(copy.deepcopy(base).cuda(), 192, 1, 16, code_positions="appended")(ids, baseline=True)["ce"]
        full = _model(["full_attention"] * 2)
        full.load_state_dict(base.state_dict())
        other = CompressLM(full.cuda(), 192, 1, 16, code_positions="appended")(ids, baseline=True)["ce"]
    assert torch.isfinite(got) and float(got) != float(other)
