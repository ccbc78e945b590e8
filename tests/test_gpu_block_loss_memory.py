"""The loss's gradient takes the memory of its elements, however far apart the logits' rows lie."""

from __future__ import annotations

import pytest
import torch

from tests.block_helpers import UNIT, close, cross_entropy64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_gradient_of_far_rows(cuda_device, dtype):
    from isa.kernels.transformer_block import cross_entropy, cross_entropy_with_grad

    g = torch.Generator(device=cuda_device).manual_seed(0)
    whole = torch.randn(6, 64, 1003, generator=g, device=cuda_device).to(dtype)
    many = torch.randn(96, 1003, generator=g, device=cuda_device).to(dtype)
    for name, x in (("last tokens", whole[:, -1]), ("every eighth row", many[::8]), ("a window of columns", many[:, 3:203]),
                    ("a padded vocabulary", many[:, :1000]), ("few classes", many[:, 5:8]),
                    ("an unaligned row", whole[:, 1, 1:])):
        print(f"[case] {name} {dtype}", flush=True)
        t = torch.randint(0, x.shape[1], x.shape[:1], generator=g, device=cuda_device)
        row, grad = cross_entropy64(x, t, -100)
        n = x.shape[0]
        loss, one = cross_entropy_with_grad(x, t)
        leaf = x.detach().requires_grad_(True)
        (two,) = torch.autograd.grad(cross_entropy(leaf, t), leaf)
        assert abs(float(loss) - float(row.mean())) <= 64 * UNIT[torch.float32] * 20
        for dx in (one, two):
            close(dx, grad / n, UNIT[dtype] + 64 * UNIT[torch.float32], "gradient")
            held = dx.untyped_storage().nbytes()
            assert held <= 1.25 * dx.numel() * dx.element_size(), (name, held, dx.numel() * dx.element_size())


def test_memory_of_a_last_tokens_loss(cuda_device):
    from isa.kernels.transformer_block import cross_entropy

    x = torch.zeros(8, 512, 50304, dtype=torch.bfloat16, device=cuda_device)  # 412 MB
    last = x[:, -1].requires_grad_(True)
    t = torch.arange(8, device=cuda_device)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    (dx,) = torch.autograd.grad(cross_entropy(last, t), last)
    assert torch.cuda.max_memory_allocated() - before <= 4 * last.numel() * 2
    assert dx.shape == last.shape
