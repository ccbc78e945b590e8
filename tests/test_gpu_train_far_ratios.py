"""The policy loss where a ratio passes fp32's largest number: rows without an advantage have no part in the loss."""

from __future__ import annotations

import math

import pytest
import torch

from tests.block_helpers import UNIT, close
from tests.train_helpers import policy64

pytestmark = pytest.mark.gpu
V = UNIT[torch.float32]


@pytest.mark.parametrize("clip", [0.2, (0.1, 0.3), None], ids=str)
@pytest.mark.parametrize("vocab", [50, 1000, 70001])
def test_no_advantage_far_from_the_old_policy(cuda_device, vocab, clip):
    """Rows 0 to 3: advantage 0 (of either sign) and l - old = 100, 88, 300 and -300; the others as ever. l is a difference of
    numbers up to 20, off by 64 v of that, and so is a ratio's exponent (ratios up to e^0.5 of advantages up to 4)."""
    from isa.kernels.transformer_block import policy_loss, policy_loss_with_grad

    print(f"[case] {vocab} {clip}", flush=True)
    g = torch.Generator(device=cuda_device).manual_seed(vocab)
    x = torch.randn(12, vocab, generator=g, device=cuda_device)
    t = torch.randint(0, vocab, (12,), generator=g, device=cuda_device)
    now = torch.log_softmax(x.double(), -1).gather(1, t[:, None])[:, 0]
    d = torch.linspace(-0.5, 0.5, 12, dtype=torch.float64, device=cuda_device)
    d[:4] = torch.tensor([100.0, 88.0, 300.0, -300.0], dtype=torch.float64, device=cuda_device)
    a = torch.randn(12, generator=g, device=cuda_device).clamp(-4.0, 4.0)
    a[:4] = torch.tensor([0.0, -0.0, -0.0, 0.0], device=cuda_device)
    old = (now - d).float()
    low, high = (1.0, math.inf) if clip is None else clip if isinstance(clip, tuple) else (clip, clip)
    row, grad, _ = policy64(x, t, old, a, None, low, min(high, 1e300), 0.0, -100)
    off = 64 * V * 20 * 8
    for reduction, want in (("mean", row.mean()), ("sum", row.sum()), ("none", row)):
        leaf = x.clone().requires_grad_(True)
        loss, _ = policy_loss(leaf, t, old, a, clip=clip, reduction=reduction)
        assert float((loss.detach().double().cpu() - want).abs().max()) <= off * (12 if reduction == "sum" else 1)
        (dx,) = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
        assert torch.count_nonzero(dx[:4]) == 0
        close(dx, grad / (12 if reduction == "mean" else 1), V + 4 * 64 * V * 20, reduction)
    loss, dx, _ = policy_loss_with_grad(x, t, old, a, clip=clip)
    assert abs(float(loss) - float(row.mean())) <= off and torch.count_nonzero(dx[:4]) == 0
    close(dx, grad / 12, V + 4 * 64 * V * 20, "one pass")


def test_what_is_not_a_number_stays(cuda_device):
    """An advantage of 0 hides neither an action outside the vocabulary nor a NaN."""
    from isa.kernels.transformer_block import policy_loss

    x, a = torch.randn(5, 50, device=cuda_device), torch.zeros(5, device=cuda_device)
    t, old = torch.tensor([1, 50, 2, 3, 4], device=cuda_device), torch.full((5,), -4.0, device=cuda_device)
    old[2] = math.nan
    x[3, 7] = math.nan
    rows, _ = policy_loss(x, t, old, a, reduction="none")
    assert torch.isnan(rows).tolist() == [False, True, True, True, False]
    assert rows[0] == 0.0 and rows[4] == 0.0
