"""On-policy distillation from a teacher's most likely tokens: sample, score, train; a few updates.

Each update samples one action per prompt from the student itself (``sample_tokens``, with exponential random numbers
that this program draws), has the teacher name its 16 most likely tokens at every sampled position
(``teacher_topk_logprobs``), and takes a step on the reverse divergence between the two
(``topk_distillation_losses``). Student and teacher are randomly initialised one-layer models.

Run ``python examples/topk_distillation.py`` (CPU fp32, or bf16 on a B200).
"""

import json
import random
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent))
sys.path.insert(1, str(Path(__file__).resolve().parents[1]))  # run from a source checkout

from _tiny_model import VOCAB_SIZE, tiny_qwen3  # noqa: E402

from thundersync_b200.engine.layers import Executor, Segment  # noqa: E402
from thundersync_b200.opd.objectives import teacher_topk_logprobs, topk_distillation_losses  # noqa: E402
from thundersync_b200.ops.gemm import gemm  # noqa: E402
from thundersync_b200.ops.sampling import sample_tokens  # noqa: E402


@torch.no_grad()
def rollout(model, prompts: list[list[int]], length: int, generator: torch.Generator):
    """``length`` sampled tokens after each prompt, and the log-probs they were drawn with: [B, length] each."""
    device = next(model.parameters()).device
    ex = Executor(model)
    # the prompts as one pack; afterwards one token of each sequence at a time, over its own K/V chunks
    new, start, segs = [t for p in prompts for t in p], 0, []
    pos = [i for p in prompts for i in range(len(p))]
    for p in prompts:
        segs.append(Segment(start, len(p), []))
        start += len(p)
    chains: list[list] = [[([], []) for _ in range(ex.spec.n_layers)] for _ in prompts]
    ids = torch.tensor(new, device=device)
    last = torch.tensor([s.start + s.length - 1 for s in segs], device=device)
    tokens, logprobs = [], []
    for step in range(length):
        h, states = ex.run(ids, torch.tensor(pos, device=device), segs)
        for chain, st in zip(chains, states):
            for (ks, vs), (k, v) in zip(chain, st):
                ks.append(k)
                vs.append(v)
        logits = gemm(h.index_select(0, last), ex.head_weight(), out_dtype=torch.float32)
        noise = torch.empty_like(logits).exponential_(generator=generator)
        ids, lp = sample_tokens(logits, noise, temperature=1.0, top_p=0.99)
        tokens.append(ids)
        logprobs.append(lp)
        pos = [len(p) + step for p in prompts]
        segs = [Segment(i, 1, [(list(ks), list(vs)) for ks, vs in chain]) for i, chain in enumerate(chains)]
        last = torch.arange(len(prompts), device=device)
    return torch.stack(tokens, 1), torch.stack(logprobs, 1)


def main():
    torch.manual_seed(3)
    device = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    student, teacher = tiny_qwen3(device).eval(), tiny_qwen3(device).eval()
    with torch.no_grad():
        teacher.lm_head.weight.mul_(8.0)  # a teacher with opinions: its random logits are otherwise nearly flat
    optimizer = torch.optim.AdamW(student.parameters(), lr=2e-3, weight_decay=0.0)
    generator = torch.Generator(device=device).manual_seed(7)
    rng = random.Random(5)
    prompts = [[rng.randrange(VOCAB_SIZE) for _ in range(rng.randint(3, 6))] for _ in range(4)]
    losses, norm, entropy = [], 0.0, 0.0
    for _ in range(10):
        actions, logprobs = rollout(student, prompts, 8, generator)
        entropy = -float(logprobs.mean())
        optimizer.zero_grad()
        total, count = 0.0, 0
        for prompt, action in zip(prompts, actions.tolist()):
            turns = [(action, [True] * len(action))]
            ids, lp = teacher_topk_logprobs(teacher, prompt, turns, 16)
            loss = topk_distillation_losses(student, prompt, turns, ids, lp, direction="reverse")
            loss.sum().backward()
            total, count = total + float(loss.detach().sum()), count + loss.numel()
        for p in student.parameters():
            if p.grad is not None:
                p.grad.div_(count)
        norm = float(torch.nn.utils.clip_grad_norm_(student.parameters(), 1.0))
        if not (norm > 0 and norm == norm):
            raise RuntimeError(f"expected a finite, nonzero gradient norm, got {norm}")
        optimizer.step()
        losses.append(total / count)
    print(json.dumps({"objective": "topk_distillation", "updates": len(losses), "gradient_norm": norm,
                      "first_loss": losses[0], "loss": losses[-1], "sampled_entropy": entropy,
                      "device": device.type}))


if __name__ == "__main__":
    main()
