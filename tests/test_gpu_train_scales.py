"""Scales of the embedding at the ends of what fp32 holds."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_scales_that_fp32_does_not_hold_are_refused(cuda_device):
    from isa.kernels.transformer_block import embedding

    w = torch.full((3, 8), 1e-30, device=cuda_device, requires_grad=True)
    ids = torch.tensor([0, 2, 2], device=cuda_device)
    for bad in (1e39, -1e39, 1e300, math.inf, -math.inf, math.nan):
        with pytest.raises(RuntimeError, match="scale must be finite"):
            embedding(ids, w, scale=bad)
    for good in (3e38, -3e38, 0.0, 1e-30):
        y = embedding(ids, w, scale=good)
        (g,) = torch.autograd.grad(y.sum(), w)
        want = good * torch.tensor([1.0, 0.0, 2.0], dtype=torch.float64)  # (twice 3e38 is past fp32, too)
        # (1e-60 is 0 in fp32, whose smallest number is 2^-149)
        torch.testing.assert_close(y[0, 0].item(), good * 1e-30, rtol=1e-6, atol=2.0 ** -149)
        torch.testing.assert_close(g[:, 0].cpu(), want.float(), rtol=1e-6, atol=0.0)
