"""The teacher's entries and the distillation loss over whole trajectories, and the example that runs them together."""

from __future__ import annotations

import json
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]
PROMPT = [3, 17, 40, 5]
TURNS = [([9, 2, 33], [False, True, True]), ([8], [False]), ([1, 60, 7, 7], [True, True, False, True])]


def _model(seed: int, device="cpu"):
    from thundersync_b200 import Qwen3Config, Qwen3ForCausalLM

    torch.manual_seed(seed)
    cfg = Qwen3Config(vocab_size=64, hidden_size=128, intermediate_size=256, num_hidden_layers=1,
                      num_attention_heads=2, num_key_value_heads=1, head_dim=64, max_position_embeddings=128,
                      tie_word_embeddings=False)
    model = Qwen3ForCausalLM(cfg).to(device)
    return model.to(torch.bfloat16 if device == "cuda" else torch.float32).eval()


def _scored_logits(model):
    from thundersync_b200.engine.layers import full_causal_logits

    toks = PROMPT + [t for tk, _ in TURNS for t in tk]
    mask = [False] * len(PROMPT) + [s for _, sc in TURNS for s in sc]
    device = next(model.parameters()).device
    z = full_causal_logits(model, torch.tensor(toks, device=device))
    return z[torch.tensor([i - 1 for i, s in enumerate(mask) if s], device=device)]


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_teacher_entries_and_loss(device):
    from thundersync_b200.opd.objectives import teacher_topk_logprobs, topk_distillation_losses

    teacher, student = _model(1, device), _model(2, device)
    ids, lp = teacher_topk_logprobs(teacher, PROMPT, TURNS, 64, temperature=1.5, rows=2)
    z = _scored_logits(teacher).double()
    want, order = torch.log_softmax(z / 1.5, -1).sort(dim=-1, descending=True, stable=True)
    assert ids.shape == (5, 64)
    # the same fp32 logits on both sides: their order is exact, the log-probs to fp32
    assert torch.equal(ids, order)
    torch.testing.assert_close(lp.double(), want, rtol=4e-7, atol=4e-6)
    loss = topk_distillation_losses(student, PROMPT, TURNS, ids, lp, temperature=1.5)
    q = torch.log_softmax(_scored_logits(student).double() / 1.5, -1).gather(-1, ids)
    p = lp.double()
    # all 64 tokens are entries: the whole divergence. The loss's own logits carry an error of 1e-6
    torch.testing.assert_close(loss.detach().double(), (p.exp() * (p - q)).sum(-1).detach(), rtol=1e-4, atol=2e-5)
    grads = torch.autograd.grad(loss.sum(), [x for x in student.parameters() if x.requires_grad])
    assert all(bool(torch.isfinite(g).all()) for g in grads) and any(float(g.abs().sum()) > 0 for g in grads)


def test_nothing_scored():
    from thundersync_b200.opd.objectives import teacher_topk_logprobs, topk_distillation_losses

    turns = [([1, 2], [False, False])]
    model = _model(1)
    ids, lp = teacher_topk_logprobs(model, PROMPT, turns, 4)
    assert tuple(ids.shape) == tuple(lp.shape) == (0, 4)
    assert topk_distillation_losses(model, PROMPT, turns, ids, lp).numel() == 0


def test_a_student_equal_to_its_teacher_has_no_gradient():
    from thundersync_b200.opd.objectives import teacher_topk_logprobs, topk_distillation_losses

    model = _model(4)
    ids, lp = teacher_topk_logprobs(model, PROMPT, TURNS, 8)
    for direction in ("forward", "reverse"):
        loss = topk_distillation_losses(model, PROMPT, TURNS, ids, lp, direction=direction)
        assert float(loss.detach().abs().max()) <= 1e-5
        (g,) = torch.autograd.grad(loss.sum(), model.lm_head.weight)
        assert float(g.abs().max()) <= 1e-4


def _run(cuda: bool) -> dict:
    env = dict(os.environ)
    if not cuda:
        env["CUDA_VISIBLE_DEVICES"] = ""
    out = subprocess.run([sys.executable, str(ROOT / "examples" / "topk_distillation.py")], env=env,
                         capture_output=True, text=True, timeout=600, check=True)
    return json.loads(out.stdout.strip().splitlines()[-1])


@pytest.mark.parametrize("cuda", [False, pytest.param(True, marks=pytest.mark.gpu)])
def test_example(cuda):
    rec = _run(cuda)
    assert rec["objective"] == "topk_distillation" and rec["gradient_norm"] > 0
    assert rec["loss"] < rec["first_loss"]  # ten steps towards the teacher
