"""Tensors of more than 2^31 elements: what lies at their far end is what the formulas give."""

from __future__ import annotations

import pytest
import torch

from tests.block_helpers import UNIT, close
from tests.train_helpers import philox, policy64, preference64

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
V = UNIT[torch.float32]


def test_many_tokens_and_a_large_table(cuda_device):
    from isa.kernels.transformer_block import embedding

    for tokens, vocab, dim in ((2_200_003, 1000, 1000), (300, 4_200_003, 520)):
        print(f"[case] {tokens} tokens of {vocab} x {dim}", flush=True)
        assert max(tokens, vocab) * dim > 2 ** 31
        w = torch.zeros(vocab, dim, dtype=BF16, device=cuda_device)
        w[-50:] = torch.randn(50, dim, device=cuda_device)
        w.requires_grad_(True)
        ids = torch.randint(0, vocab - 50, (tokens,), device=cuda_device)
        ids[-20:] = vocab - 1 - torch.arange(20, device=cuda_device)
        y = embedding(ids, w)
        assert torch.equal(y[-20:], w.detach()[ids[-20:]])
        dy = torch.zeros_like(y)
        dy[-20:] = torch.randn(20, dim, device=cuda_device)
        (dw,) = torch.autograd.grad(y, w, dy)
        assert torch.equal(dw[ids[-20:]], dy[-20:])
        assert torch.count_nonzero(dw[:-20]) == 0
        del y, dy, dw, w


def test_dropout_of_many_elements(cuda_device):
    from isa.kernels.transformer_block import dropout, dropout_add_layer_norm

    for rows, dim in ((2 ** 21 + 3, 1024), (2 ** 21 + 3, 1025)):
        print(f"[case] dropout {rows} x {dim}", flush=True)
        seed = torch.tensor([11, 12], device=cuda_device)
        x = torch.ones(rows, dim, dtype=BF16, device=cuda_device)
        y = dropout(x, 0.5, seed)
        groups = -(-dim // 8)
        for r in (0, rows - 1):
            kept = []
            for g in range(r * groups, (r + 1) * groups):
                words = philox((g & 0xFFFFFFFF, g >> 32, 12, 0), (11, 0))
                kept += [(w >> s) & 0xFFFF for w in words for s in (0, 16)]
            want = (torch.tensor(kept[:dim]) >= 32768).double() * 2.0
            assert torch.equal(y[r].double().cpu(), want), r
        if dim == 1024:
            _, h = dropout_add_layer_norm(x, torch.zeros_like(x), torch.ones(dim, dtype=BF16, device=cuda_device), p=0.5, seed=seed)
            assert torch.equal(h, y)
            del h
        del x, y


def test_losses_of_many_logits(cuda_device):
    from isa.kernels.transformer_block import policy_loss_with_grad, preference_loss_with_grad

    rows, vocab = 43000, 50304
    assert rows * vocab > 2 ** 31
    x = torch.zeros(rows, vocab, dtype=BF16, device=cuda_device)
    x[-3:] = torch.randn(3, vocab, device=cuda_device) * 2.0
    t = torch.full((rows,), -100, device=cuda_device)
    t[-3:] = torch.tensor([5, vocab - 1, 777], device=cuda_device)
    f = torch.zeros(rows, device=cuda_device)
    f[-3:] = torch.tensor([1.0, -0.5, 2.0], device=cuda_device)
    old = f - 12.0
    loss, dx, logp = policy_loss_with_grad(x, t, old, f, clip=None)
    row, grad, l = policy64(x[-3:], t[-3:], old[-3:], f[-3:], None, 1.0, float("inf"), 0.0, -100)
    assert abs(float(loss) - float(row.mean())) <= 256 * V * 20 * float(row.abs().max())
    close(dx[-3:], grad / 3, UNIT[BF16] + 64 * V * 20, "policy gradient")
    assert torch.count_nonzero(dx[:-3]) == 0 and torch.count_nonzero(logp[:-3]) == 0
    del dx
    ref = torch.tensor([-1.0, -30.0], device=cuda_device)
    loss, dx, logp = preference_loss_with_grad(x.view(2, rows // 2, vocab), t.view(2, -1), ref)
    # the chosen sequence has no token that counts
    small = torch.zeros(2, 3, vocab, dtype=BF16, device=cuda_device)
    small[1] = x[-3:]
    u = torch.full((2, 3), -100, device=cuda_device)
    u[1] = t[-3:]
    want, grad, total = preference64(small, u, ref, 0.1, -100)
    assert abs(float(loss) - float(want[0])) <= 64 * V * 60 and abs(float(logp[1]) - float(total[1])) <= 64 * V * 60
    close(dx[1, -3:], grad[1], UNIT[BF16] + 64 * V * 20, "preference gradient")
    assert torch.count_nonzero(dx[0]) == 0 and torch.count_nonzero(dx[1, :-3]) == 0
