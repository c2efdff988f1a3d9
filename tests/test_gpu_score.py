"""The operators on logits as a model uses them, on a B200: ``BDH.score`` against torch's log softmax
of the same logits in 64 bits, and the distillation example (teacher's lists, student's loss, scores)."""

import importlib.util

import pytest
import torch

import bdh_model
from conftest import REPO

pytestmark = pytest.mark.gpu


def _model(**kw):
    torch.manual_seed(0)
    cfg = bdh_model.BDHConfig(n_layer=2, n_embd=64, n_head=4, mlp_internal_dim_multiplier=8, dropout=0.0, **kw)
    return bdh_model.BDH(cfg).cuda().eval()


@pytest.mark.parametrize("vocab", [256, 300])
@pytest.mark.parametrize("amp", [None, torch.bfloat16])
def test_score_is_the_log_softmax_of_the_models_logits(monkeypatch, amp, vocab):
    monkeypatch.setenv("BDH_ATTN_IMPL", "cuda_sm100")
    m = _model(vocab_size=vocab)
    idx = torch.randint(vocab, (3, 90), device="cuda")
    idx[1, 40:] = -100
    with torch.autocast("cuda", dtype=amp or torch.bfloat16, enabled=amp is not None):
        r = m.score(idx, top_k=5, temperature=0.8)
        logits = m(idx.masked_fill(idx == -100, 0))[0].detach()
    assert logits.dtype == (amp or torch.float32)
    z = logits[:, :-1].double() / 0.8
    lp = torch.log_softmax(z, -1)
    want = torch.where(idx[:, 1:] == -100, 0.0, lp.gather(-1, idx[:, 1:].clamp_min(0).unsqueeze(-1))[..., 0])
    assert (r.logprob - want).abs().max().item() < 2e-5  # |z| < 10: roundings of 1e-6
    assert (r.entropy - torch.special.entr(lp.exp()).sum(-1)).abs().max().item() < 5e-5
    order = torch.sort(logits[:, :-1], dim=-1, descending=True, stable=True)
    assert torch.equal(r.top_index, order.indices[..., :5])
    assert not r.logprob.requires_grad


def test_distillation_example_runs_and_learns(monkeypatch):
    monkeypatch.setenv("BDH_ATTN_IMPL", "cuda_sm100")
    spec = importlib.util.spec_from_file_location("distill_top_lists", REPO / "examples" / "distill_top_lists.py")
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    out = ex.main(["--steps", "40", "--batch", "8", "--length", "96"])
    assert out["student_bits_before"] > 7.5  # an untrained byte model knows nothing: 8 bits
    assert out["student_bits"] < 5.5         # letters and spaces alone: log2(27) = 4.75 if all were as frequent
    assert 0.0 <= out["last_loss"] < 0.6 * out["first_loss"]
