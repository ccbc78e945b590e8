"""The loss takes as many rows as the library says it does (2^24): a launch of a block a row has more
threads than one dimension of a grid may hold."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [(1 << 24) - 3, 1 << 24])
def test_most_rows(cuda_device, rows):
    """Rows of one kind each, whose losses are known: log(1 + 3 e^-x) for logits x, 0, 0, 0 and the first target."""
    from isa.kernels.transformer_block import cross_entropy, cross_entropy_with_grad

    print(f"[case] {rows} rows", flush=True)
    x = torch.zeros(rows, 4, dtype=torch.bfloat16, device=cuda_device)
    x[:, 0] = (torch.arange(rows, device=cuda_device) % 7).to(torch.bfloat16)
    t = torch.zeros(rows, dtype=torch.int64, device=cuda_device)
    t[::5] = -100
    want = torch.log1p(3.0 * torch.exp(-torch.arange(7.0, dtype=torch.float64, device=cuda_device)))
    each = want[torch.arange(rows, device=cuda_device) % 7]
    got = cross_entropy(x, t, reduction="none")
    assert float((got.double() - each * (t == 0)).abs().max()) <= 64 * 2.0 ** -24
    mean = float(each[t == 0].mean())
    loss, dx = cross_entropy_with_grad(x, t, grad_scale=float(rows))
    assert abs(float(loss) - mean) <= 2.0 ** -12 * mean  # 2^14 terms a thread in fp32
    p = torch.exp(-each).unsqueeze(1)
    first = (p - 1.0) * (t == 0).unsqueeze(1) * (rows / int((t == 0).sum()))
    assert float((dx[:, :1].double() - first).abs().max()) <= 2.0 ** -8
    leaf = x.requires_grad_(True)
    loss = cross_entropy(leaf, t, reduction="sum")
    (dy,) = torch.autograd.grad(loss, leaf)
    assert abs(float(loss) - mean * int((t == 0).sum())) <= 2.0 ** -12 * float(loss)
    assert float((dy[:, :1].double() - (p - 1.0) * (t == 0).unsqueeze(1)).abs().max()) <= 2.0 ** -8
