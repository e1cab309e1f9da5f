"""Every loss of the training wrapper that names a cross entropy, with ``fused_ce`` and without."""
import copy

import pytest
import torch

from test_gpu_gate import _model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["per token", "teacher logits", "masked teacher logits", "self-teacher", "frozen teacher",
                                  "frozen teacher in chunks"])
def test_cross_entropies_are_the_fused_ones(kind, monkeypatch):
    """The same logits, so the losses differ by fp32 sums alone (1e-5 of ~5.6) and the gradients by that and the rounding of the
    logits' gradients to bf16 (2^-8 of each, at random: 2^-8 of the norm; where two losses share the logits, each is rounded and
    their sum: three times that). The library's cross entropy is not called."""
    from abridgekv_amd import compress_forward as cf
    base = _model(44)
    gen = torch.Generator().manual_seed(1)
    ids = torch.randint(0, 257, (2, 3, 64), generator=gen).cuda()
    mask = torch.ones((2, 3, 64), device="cuda")
    mask[0, 0, :40] = 0
    rows = 2 * 3 * 63
    teacher = torch.randn((rows, 257), generator=gen).cuda()
    hidden = torch.randn((rows, base.config.hidden_size), generator=gen).to(torch.bfloat16).cuda()
    kw = {"per token": {"resp_mask": mask, "per_token": True},
          "teacher logits": {"distill_lambda": 0.5, "teacher_logits": teacher, "distill_temp": 2.0},
          "masked teacher logits": {"resp_mask": mask, "teacher_logits": teacher},
          "self-teacher": {"distill_lambda": 0.5},
          "frozen teacher": {"resp_mask": mask, "teacher_rows": hidden},
          "frozen teacher in chunks": {"resp_mask": mask, "teacher_rows": hidden, "ce_chunk": 100, "distill_temp": 1.5}}[kind]
    res, grads = [], []
    for fused_ce in (False, True):
        torch.manual_seed(0)
        clm = cf.CompressLM(copy.deepcopy(base).cuda(), 64, 3, 16, code_positions="bitrev", fused_ce=fused_ce)
        if "teacher_rows" in kw:
            kw["teacher_head"] = copy.deepcopy(clm.model.lm_head)
        calls, real = [], torch.nn.functional.cross_entropy
        monkeypatch.setattr(cf.F, "cross_entropy", lambda *a, **k: (calls.append(1), real(*a, **k))[1])
        out = clm(ids, **kw)
        monkeypatch.undo()
        assert bool(calls) != fused_ce
        (out["ce_pt"].mean() if "ce_pt" in out else out["ce"] + out["distill"]).backward()
        res.append(out)
        grads.append(clm.model.lm_head.weight.grad.double())
    for name, a in res[0].items():
        assert torch.allclose(a.double(), res[1][name].double(), atol=1e-5, rtol=1e-5), name
    assert (grads[0] - grads[1]).norm() <= 3 * 2.0 ** -8 * grads[0].norm()
