"""Distillation of a small BDH from a larger one's top lists, and the student's score on held-out bytes.

    python examples/distill_top_lists.py [--steps 200] [--top 16] [--temperature 2.0]

The teacher (a byte model, first trained for a few steps on the same text) reads the training text once and
keeps, for every position, the log probabilities of its ``--top`` most probable next bytes
(``kernels.token_logprobs``): 192 bytes a position instead of 1 KB of logits, and for a vocabulary of 131072
instead of 512 KB. The student is trained on those lists alone (``kernels.distill_topk_loss``, the probability
outside a list as one more class), and both are scored on held-out text (``BDH.score``).

The text is synthetic: words drawn from a small vocabulary of random bytes. Needs a B200.
"""

from __future__ import annotations

import argparse
import os
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "bdh-gpu-fast_b200"))

import torch

import kernels
from bdh_model import BDH, BDHConfig

os.environ.setdefault("BDH_ATTN_IMPL", "cuda_sm100")


def text(n: int, seed: int) -> torch.Tensor:
    g = torch.Generator().manual_seed(seed)
    words = [torch.randint(97, 123, (int(k),), generator=torch.Generator().manual_seed(i))
             for i, k in enumerate(torch.randint(2, 8, (50,), generator=torch.Generator().manual_seed(0)))]
    out = []
    while sum(len(w) + 1 for w in out) < n:
        out.append(words[int(torch.randint(50, (1,), generator=g))])
    return torch.cat([torch.cat([w, torch.tensor([32])]) for w in out])[:n]


def batches(data: torch.Tensor, batch: int, length: int) -> torch.Tensor:
    n = data.numel() // (batch * length) * batch * length
    return data[:n].view(-1, batch, length)


def train_teacher(model: BDH, data: torch.Tensor, steps: int, lr: float) -> None:
    opt = torch.optim.AdamW(model.parameters(), lr=lr)
    for step in range(steps):
        idx = data[step % len(data)]
        r = kernels.token_logprobs(model(idx[:, :-1])[0], idx[:, 1:])  # (the targets' log probabilities)
        loss = -r.logprob.mean()
        opt.zero_grad()
        loss.backward()
        opt.step()


def teacher_lists(model: BDH, data: torch.Tensor, top: int, temperature: float):
    with torch.inference_mode():
        return [model.score(idx, top_k=top, temperature=temperature) for idx in data]


def distill(student: BDH, data: torch.Tensor, lists, steps: int, temperature: float, lr: float):
    opt = torch.optim.AdamW(student.parameters(), lr=lr)
    losses = []
    for step in range(steps):
        idx, top = data[step % len(data)], lists[step % len(data)]
        logits = student(idx)[0][:, :-1]
        weight = torch.full((), temperature ** 2 / top.lse.numel(), device=idx.device)
        loss = kernels.distill_topk_loss(logits, top.top_index, top.top_logprob, weight=weight,
                                         temperature=temperature, tail=True).sum()
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


def bits_per_byte(model: BDH, data: torch.Tensor) -> float:
    with torch.inference_mode():
        return -torch.stack([model.score(idx).logprob.mean() for idx in data]).mean().item() / 0.6931471805599453


def main(argv=None) -> dict:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--top", type=int, default=16)
    ap.add_argument("--temperature", type=float, default=2.0)
    ap.add_argument("--batch", type=int, default=16)
    ap.add_argument("--length", type=int, default=128)
    ap.add_argument("--lr", type=float, default=2e-3)
    a = ap.parse_args(argv)
    torch.manual_seed(0)
    data = batches(text(8 * a.batch * a.length, 1), a.batch, a.length).cuda()
    held = batches(text(2 * a.batch * a.length, 2), a.batch, a.length).cuda()
    teacher = BDH(BDHConfig(n_layer=3, n_embd=128, n_head=4, mlp_internal_dim_multiplier=16, dropout=0.0)).cuda()
    student = BDH(BDHConfig(n_layer=1, n_embd=64, n_head=4, mlp_internal_dim_multiplier=16, dropout=0.0)).cuda()
    train_teacher(teacher, data, a.steps, a.lr)
    lists = teacher_lists(teacher, data, a.top, a.temperature)
    before = bits_per_byte(student, held)
    losses = distill(student, data, lists, a.steps, a.temperature, a.lr)
    out = {"teacher_bits": bits_per_byte(teacher, held), "student_bits_before": before,
           "student_bits": bits_per_byte(student, held), "first_loss": losses[0], "last_loss": losses[-1]}
    print("  ".join(f"{k} {v:.4f}" for k, v in out.items()))
    return out


if __name__ == "__main__":
    main()
