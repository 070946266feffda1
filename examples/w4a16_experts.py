"""Quantize the experts of an MoE layer to int4 with GPTQ and serve them on the 4-bit weights.

The calibration tokens go through the experts as the router sends them; the solve is
batched over the experts; the served layer reads the packed codes.

    python examples/w4a16_experts.py --experts 64 --hidden 2048 --intermediate 768 --tokens 8192
"""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "llm-compressor_amd"))

from llmcompressor_amd import GPTQModifier, W4A16Experts  # noqa: E402
from llmcompressor_amd.moe import LinearExperts  # noqa: E402


class MoELayer(torch.nn.Module):
    def __init__(self, experts: int, top: int, hidden: int, intermediate: int, g: torch.Generator, device):
        super().__init__()
        shapes = (experts, intermediate, hidden), (experts, intermediate, hidden), (experts, hidden, intermediate)
        self.experts = LinearExperts.from_stacked(*(
            (torch.randn(s, generator=g, device=device) * 0.02).to(torch.bfloat16) for s in shapes))
        self.experts.sorted_tokens = True
        self.register_buffer("router", torch.randn(experts, hidden, generator=g, device=device) * 0.05)
        self.top = top

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        weights, ids = torch.softmax(x.float() @ self.router.t(), -1).topk(self.top)
        return self.experts(x, ids, weights / weights.sum(-1, keepdim=True))


def serve(experts: int, top: int, hidden: int, intermediate: int, tokens: int, seed: int = 0, device="cuda"):
    """Relative errors against the bf16 layer's output: of the quantized layer, and of the served one."""
    g = torch.Generator(device=device).manual_seed(seed)
    layer = MoELayer(experts, top, hidden, intermediate, g, device)
    x = torch.randn(tokens, hidden, generator=g, device=device).to(torch.bfloat16)
    with torch.no_grad():
        want = layer(x).float()
        GPTQModifier(scheme="W4A16").apply(layer, [x])
        quantized = layer(x).float()
        layer.experts = W4A16Experts.from_experts(layer.experts)
        served = layer(x).float()
    return tuple(float((y - want).norm() / want.norm()) for y in (quantized, served))


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, default in (("experts", 64), ("top", 8), ("hidden", 2048), ("intermediate", 768), ("tokens", 8192)):
        ap.add_argument(f"--{name}", type=int, default=default)
    errors = serve(**vars(ap.parse_args()))
    print(f"relative error: quantized {errors[0]:.4f}, served on 4-bit weights {errors[1]:.4f}")
