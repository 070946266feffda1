"""Train a pruned gated MLP in block-scaled fp8 towards its dense bf16 original.

Half of the MLP's weights (the smallest of each) are set to zero, and a few
steps of distillation train what is there in fp8: e4m3 weights with a scale per
128 x 128 block, quantized anew from fp32 masters in every step, every product on
fp8 codes, the backward pass from 8-bit checkpoints of the activations.

    python examples/fp8_mlp_recovery.py --hidden 2048 --intermediate 768 --tokens 4096 --steps 20
"""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "llm-compressor_amd"))

from llmcompressor_amd import Fp8GatedMLP  # noqa: E402
from llmcompressor_amd.moe import ExpertMLP  # noqa: E402


def recover(hidden: int, intermediate: int, tokens: int, steps: int, lr: float = 1e-3, seed: int = 0, device="cuda"):
    """Relative error of the student's output against the teacher's, before each step and after the last."""
    g = torch.Generator(device=device).manual_seed(seed)
    teacher = ExpertMLP(hidden, intermediate, dtype=torch.bfloat16, device=device)
    with torch.no_grad():
        for p in teacher.parameters():
            p.copy_(torch.randn(p.shape, generator=g, device=device) * 0.02)
    student = Fp8GatedMLP.from_expert(teacher, trainable=True).float()   # fp32 masters for the optimiser
    with torch.no_grad():
        for p in student.parameters():
            p.masked_fill_(p.abs() < p.abs().median(), 0.0)
    optimiser = torch.optim.Adam(student.parameters(), lr=lr)
    x = torch.randn(tokens, hidden, generator=g, device=device).to(torch.bfloat16)
    with torch.no_grad():
        want = teacher(x).float()

    def error():
        with torch.no_grad():
            return float((student(x).float() - want).norm() / want.norm())

    errors = [error()]
    for _ in range(steps):
        optimiser.zero_grad(set_to_none=True)
        loss = (student(x).float() - want).square().sum(1).mean()
        loss.backward()
        optimiser.step()
        errors.append(error())
    return errors


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, default in (("hidden", 2048), ("intermediate", 768), ("tokens", 4096), ("steps", 20)):
        ap.add_argument(f"--{name}", type=int, default=default)
    ap.add_argument("--lr", type=float, default=1e-3)
    a = ap.parse_args()
    for i, e in enumerate(recover(a.hidden, a.intermediate, a.tokens, a.steps, a.lr)):
        print(f"step {i:3d}  relative error {e:.4f}", flush=True)
