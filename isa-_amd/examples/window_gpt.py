"""A small GPT with physical FFNs, window attention and sinks: trained to repeat what stood some
tokens before, then asked to go on, a token at a time over its cache.

    python isa-_amd/examples/window_gpt.py [--steps 150]
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import torch
import torch.nn as nn

from isa.device_models.config import make_flash_transistor_ekv_config
from isa.kernels.transformer_block import cross_entropy_with_grad
from isa.operators.block import GPT, Block, WindowAttention
from isa.operators.cim import PhysicalFFN

VOCAB, PERIOD, LENGTH, DIM = 64, 12, 96, 128


def make_model(layers: int = 2, heads: int = 4, kv_heads: int = 2, window: int = 32, sinks: int = 4) -> GPT:
    cfg = make_flash_transistor_ekv_config(default_lut_size=4096)
    blocks = nn.ModuleList(Block(DIM, WindowAttention(DIM, heads, kv_heads=kv_heads, window=window, sinks=sinks),
                                 PhysicalFFN(DIM, 2 * DIM, cfg)) for _ in range(layers))
    for block in blocks:  # gains that bring the currents of untrained thresholds to a fraction of a volt
        block.ffn.fc1.set_r_tia(2e6)
        block.ffn.fc2.set_r_tia(2e6)
    return GPT(VOCAB, 4 * LENGTH, DIM, blocks).cuda()


def batch(n: int, length: int, generator: torch.Generator) -> torch.Tensor:
    """Sequences [n, length] that repeat a random phrase of PERIOD tokens."""
    phrase = torch.randint(0, VOCAB, (n, PERIOD), generator=generator, device="cuda")
    return phrase.repeat(1, -(-length // PERIOD))[:, :length]


def train(model: GPT, steps: int, generator: torch.Generator) -> list:
    """Losses of `steps` steps. The loss gives the logits' gradient in the same pass, which the
    backward pass starts from; targets in the first phrase cannot be known and are ignored."""
    optimizer = torch.optim.AdamW(model.parameters(), lr=3e-3, weight_decay=0.0)
    losses = []
    for _ in range(steps):
        ids = batch(32, LENGTH + 1, generator)
        targets = ids[:, 1:].clone()
        targets[:, : PERIOD - 1] = -100
        optimizer.zero_grad(set_to_none=True)
        logits = model(ids[:, :-1])
        loss, gradient = cross_entropy_with_grad(logits, targets)
        logits.backward(gradient)
        optimizer.step()
        for block in model.blocks:
            block.ffn.clamp_vth()
        losses.append(loss)
    return [float(x) for x in losses]


@torch.no_grad()
def generate(model: GPT, prompt: torch.Tensor, tokens: int):
    """(the prompt and `tokens` more, the logits they were picked from)."""
    caches = model.caches(prompt.shape[0], prompt.shape[1] + tokens)
    ids, logits = [prompt], []
    step = prompt
    for _ in range(tokens):
        logits.append(model(step, caches)[:, -1])
        step = logits[-1].argmax(-1, keepdim=True)
        ids.append(step)
    return torch.cat(ids, 1), torch.stack(logits, 1)


def main() -> int:
    parser = argparse.ArgumentParser(description=__doc__)
    parser.add_argument("--steps", type=int, default=150)
    args = parser.parse_args()
    torch.manual_seed(0)
    generator = torch.Generator(device="cuda").manual_seed(0)
    model = make_model()
    losses = train(model, args.steps, generator)
    print(f"loss: first step {losses[0]:.3f}, last {losses[-1]:.3f}")
    whole = batch(4, LENGTH, generator)
    ids, _ = generate(model, whole[:, : 2 * PERIOD], LENGTH - 2 * PERIOD)
    right = (ids[:, 2 * PERIOD:] == whole[:, 2 * PERIOD:]).float().mean()
    print(f"generated tokens that repeat the phrase: {100.0 * float(right):.0f}%")
    return 0


if __name__ == "__main__":
    sys.exit(main())
