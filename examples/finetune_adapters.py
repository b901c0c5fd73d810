"""Trains low-rank adapters of a frozen transition for several tasks at once and serves them in one batch.

Each request of a batch belongs to a task and is trained with that task's adapter, the update dropped by whole rows of the pair
tensor before it joins the residual stream.  Served without dropout, all tasks share the transition's weights; a single task's
adapter can be added to them for the inference layer.

    python examples/finetune_adapters.py [--tokens 64] [--steps 200]
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import bionemo_inference_runtime_b200 as b200  # noqa: E402


def finetune(tokens: int, steps: int, tasks: int = 3, dim: int = 128, hidden: int = 512, rank: int = 8, lr: float = 1e-2):
    """Returns the losses of the steps, the student, and how far the adapted batch is from each task's own inference layer."""
    torch.manual_seed(0)
    student = b200.TrainableTransition(dim, hidden, device="cuda", dropout=0.1, dropout_shared=1, adapter_rank=rank, adapters=tasks)
    teachers = [b200.TrainableTransition(dim, hidden, device="cuda") for _ in range(tasks)]
    with torch.no_grad():  # a task is the student with other weights
        for teacher in teachers:
            own = dict(student.named_parameters())
            for name, p in teacher.named_parameters():
                p.copy_(own[name] + 0.1 * own[name].float().std().nan_to_num(0.1) * torch.randn_like(p))
    trained = [p for p in student.parameters() if p.requires_grad]
    master = [p.detach().float() for p in trained]  # the optimiser's 32-bit weights
    optimiser = torch.optim.Adam(master, lr=lr)
    index = torch.arange(2 * tasks, device="cuda", dtype=torch.int32) % tasks
    losses = []
    for _ in range(steps):
        z = torch.randn(2 * tasks, tokens, tokens, dim, device="cuda").bfloat16()
        with torch.no_grad():
            want = torch.stack([teachers[i % tasks](one, residual=True) for i, one in enumerate(z)])
        loss = (student(z, residual=True, index=index).float() - want.float()).square().mean()
        student.zero_grad()
        loss.backward()
        for m, p in zip(master, trained, strict=True):
            m.grad = p.grad.float()
        optimiser.step()
        with torch.no_grad():
            for m, p in zip(master, trained, strict=True):
                p.copy_(m)
        losses.append(loss.item())
    student.eval()
    apart = []
    with torch.no_grad():
        z = torch.randn(tasks, tokens, tokens, dim, device="cuda").bfloat16()
        together = student(z, residual=True, index=index[:tasks])
        for task in range(tasks):
            served = b200.Transition(dim, hidden, dtype=torch.bfloat16)
            served.load_state_dict(student.merged_state_dict(task), strict=True)
            apart.append((served.cuda()(z[task:task + 1], residual=True).float() - together[task].float()).abs().max().item())
    return losses, student, apart


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--tokens", type=int, default=64)
    ap.add_argument("--steps", type=int, default=200)
    a = ap.parse_args()
    losses, _, apart = finetune(a.tokens, a.steps)
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f}; the tasks' own layers differ by at most {max(apart):.4f}")
