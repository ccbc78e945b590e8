"""Operands without elements are taken whatever strides their views have."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_empty_operands_of_odd_strides(cuda_device, dtype):
    from isa.kernels.transformer_block import window_attention

    odd = torch.randn(3, 7, 4, 67, device=cuda_device).to(dtype)[..., 1:65]  # rows that no 16 bytes divide
    for name, q, k in (("no keys", odd, odd[:, :0, :2]), ("no queries", odd[:, :0], odd[:, :, :2]),
                       ("no sequences", odd[:0], odd[:0, :, :2])):
        print(f"[case] {name} {dtype}", flush=True)
        leaves = [t.detach().requires_grad_(True) for t in (q, k, k)]
        out = window_attention(*leaves, window=3, sinks=1)
        assert out.shape == q.shape and torch.count_nonzero(out) == 0
        for g, t in zip(torch.autograd.grad(out, leaves, torch.ones_like(out)), leaves):
            assert g.shape == t.shape and torch.count_nonzero(g) == 0
