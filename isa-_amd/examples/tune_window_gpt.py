"""The small GPT of window_gpt.py, tuned after its training: by rewards of its own samples (clipped policy loss with a
KL term against the model as it was), then by pairs of a right and a wrong continuation (preference loss).

    python isa-_amd/examples/tune_window_gpt.py [--steps 150] [--rounds 4]
"""

from __future__ import annotations

import argparse
import copy
import sys

import torch

from window_gpt import LENGTH, PERIOD, VOCAB, batch, generate, make_model, train

from isa.kernels.transformer_block import cross_entropy, policy_loss_with_grad, preference_loss_with_grad

PROMPT = 2 * PERIOD


def targets_of(ids: torch.Tensor) -> torch.Tensor:
    """What each token should be followed by; prompts and the last token count nowhere."""
    targets = torch.roll(ids, -1, 1)
    targets[:, : PROMPT - 1] = -100
    targets[:, -1] = -100
    return targets


@torch.no_grad()
def log_probabilities(model, ids: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
    return -cross_entropy(model(ids), targets, reduction="none")


def policy_step(model, reference, optimizer, generator: torch.Generator):
    """One round: samples, their rewards (the share of tokens that repeat the phrase) against the mean, two steps.
    Returns (mean reward, losses)."""
    whole = batch(16, LENGTH // 2, generator)
    ids, logits = generate(model, whole[:, :PROMPT], whole.shape[1] - PROMPT)
    noise = torch.rand(logits.shape, generator=generator, device=ids.device).clamp_(1e-9, 1.0 - 1e-7)
    ids[:, PROMPT:] = (logits - torch.log(-torch.log(noise))).argmax(-1)  # a sample beside each greedy choice
    targets = targets_of(ids)
    reward = (ids[:, PROMPT:] == whole[:, PROMPT:]).float().mean(1)
    advantages = (reward - reward.mean())[:, None].expand(targets.shape)
    old, ref = (log_probabilities(m, ids, targets) for m in (model, reference))
    losses = []
    for _ in range(2):
        optimizer.zero_grad(set_to_none=True)
        logits = model(ids)
        loss, gradient, _ = policy_loss_with_grad(logits, targets, old, advantages, ref_logp=ref, clip=(0.2, 0.28), kl=0.02)
        logits.backward(gradient)
        optimizer.step()
        losses.append(float(loss))
    return float(reward.mean()), losses


def preference_step(model, reference, optimizer, generator: torch.Generator) -> float:
    """One step on pairs: sequences that go on with their phrase, and the same with other tokens behind the prompt."""
    chosen = batch(8, LENGTH // 2, generator)
    rejected = chosen.clone()
    rejected[:, PROMPT:] = torch.randint(0, VOCAB, rejected[:, PROMPT:].shape, generator=generator, device=chosen.device)
    ids = torch.cat([chosen, rejected])
    targets = targets_of(ids)
    ref = log_probabilities(reference, ids, targets).sum(1)
    optimizer.zero_grad(set_to_none=True)
    logits = model(ids)
    loss, gradient, _ = preference_loss_with_grad(logits, targets, ref, beta=0.05)
    logits.backward(gradient)
    optimizer.step()
    return float(loss)


def main() -> int:
    parser = argparse.ArgumentParser(description=__doc__)
    parser.add_argument("--steps", type=int, default=150)
    parser.add_argument("--rounds", type=int, default=4)
    args = parser.parse_args()
    torch.manual_seed(0)
    generator = torch.Generator(device="cuda").manual_seed(0)
    model = make_model(dropout=0.05)
    train(model, args.steps, generator)
    model.eval()
    reference = copy.deepcopy(model).requires_grad_(False)
    optimizer = torch.optim.AdamW(model.parameters(), lr=1e-4, weight_decay=0.0)
    for i in range(args.rounds):
        reward, losses = policy_step(model, reference, optimizer, generator)
        print(f"round {i}: reward {reward:.3f}, policy losses {losses}")
    for i in range(args.rounds):
        print(f"pairs {i}: preference loss {preference_step(model, reference, optimizer, generator):.4f}")
    return 0


if __name__ == "__main__":
    sys.exit(main())
