"""Fine-tunes a transition and serves the result.

A trainable transition learns to reproduce another one from its inputs and outputs, with the residual stream of a pair
tensor as data; its weights are then loaded into the inference layer, which folds them and runs as one kernel.

    python examples/finetune_transition.py [--tokens 64] [--steps 200]
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import bionemo_inference_runtime_b200 as b200  # noqa: E402


def finetune(tokens: int, steps: int, dim: int = 128, hidden: int = 512, lr: float = 2e-3):
    """Returns the losses of the steps and the largest difference between the trained and the served layer's outputs."""
    torch.manual_seed(0)
    teacher, student = (b200.TrainableTransition(dim, hidden, device="cuda") for _ in range(2))
    with torch.no_grad():  # start near the teacher, as fine-tuning does
        for p, q in zip(student.parameters(), teacher.parameters(), strict=True):
            p.copy_(q + 0.3 * q.float().std().nan_to_num(0.1) * torch.randn_like(q))
    master = [p.detach().float() for p in student.parameters()]  # the optimiser's 32-bit weights
    optimiser = torch.optim.Adam(master, lr=lr)
    losses = []
    for _ in range(steps):
        z = torch.randn(1, tokens, tokens, dim, device="cuda").bfloat16()
        with torch.no_grad():
            want = teacher(z, residual=True)
        loss = (student(z, residual=True).float() - want.float()).square().mean()
        student.zero_grad()
        loss.backward()
        for m, p in zip(master, student.parameters(), strict=True):
            m.grad = p.grad.float()
        optimiser.step()
        with torch.no_grad():
            for m, p in zip(master, student.parameters(), strict=True):
                p.copy_(m)
        losses.append(loss.item())
    served = b200.Transition(dim, hidden, dtype=torch.bfloat16)
    served.load_state_dict(student.state_dict(), strict=True)
    with torch.no_grad():
        z = torch.randn(1, tokens, tokens, dim, device="cuda").bfloat16()
        apart = (served.cuda()(z, residual=True).float() - student(z, residual=True).float()).abs().max().item()
    return losses, apart


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--tokens", type=int, default=64)
    ap.add_argument("--steps", type=int, default=200)
    a = ap.parse_args()
    losses, apart = finetune(a.tokens, a.steps)
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f}; served layer differs by at most {apart:.4f}")
