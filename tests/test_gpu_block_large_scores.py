"""Scores of any finite size: a row's weights depend on their differences alone, so the key of the highest
score keeps weight 1 and equal ones share it, also where a score times scale log2 e passes 2^24 and
its rounding would be a power of two of its own."""

from __future__ import annotations

import pytest
import torch

from tests.block_helpers import UNIT, close

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
# of q . k: past 2^24, and as far as the types go with head_dim 64
SIZES = {torch.float32: (1e8, 1e10, 1e12, 1e20, 1e32), torch.bfloat16: (1e8, 1e10, 1e12, 1e20, 1e32),
         torch.float16: (1e8, 1e10, 1e11)}


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_equal_large_scores(cuda_device, dtype, sign):
    """All keys alike: each query's result is the mean of the values it sees."""
    from isa.kernels.transformer_block import window_attention

    g = torch.Generator(device=cuda_device).manual_seed(1)
    for size in SIZES[dtype]:
        for m, n in ((1, 1), (1, 20), (1, 700), (5, 700), (90, 90)):
            print(f"[case] {m} of {n} keys, scores {sign * size} {dtype}", flush=True)
            each = (size / 64.0) ** 0.5 * 1.1
            q = torch.full((2, m, 2, 64), each, device=cuda_device).to(dtype)
            k = torch.full((2, n, 1, 64), sign * each, device=cuda_device).to(dtype)
            v = torch.randn(2, n, 1, 64, generator=g, device=cuda_device).to(dtype)
            got = window_attention(q, k, v)
            count = torch.arange(n - m + 1, n + 1, device=cuda_device).double()[None, :, None, None]
            want = (v.double().cumsum(1)[:, n - m:] / count).expand(2, m, 2, 64)
            # equal weights are exact; the sum of n values in fp32, and one rounding
            close(got, want, UNIT[dtype] + 64 * UNIT[torch.float32], "out")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_one_large_score(cuda_device, dtype):
    """One key's score lies far above the others': the result is its value. Then far below: it has no part."""
    from isa.kernels.transformer_block import window_attention

    g = torch.Generator(device=cuda_device).manual_seed(2)
    for size in SIZES[dtype]:
        for m, n, at in ((1, 20, 3), (1, 700, 650), (90, 90, 0)):
            print(f"[case] {m} of {n} keys, one of score {size} {dtype}", flush=True)
            each = (size / 64.0) ** 0.5
            q = torch.full((1, m, 2, 64), each, device=cuda_device).to(dtype)
            k = (torch.randn(1, n, 1, 64, generator=g, device=cuda_device) / each).to(dtype)
            v = torch.randn(1, n, 1, 64, generator=g, device=cuda_device).to(dtype)
            k[:, at] = each
            got = window_attention(q, k, v)
            assert torch.equal(got, v[:, at:at + 1].expand(1, m, 2, 64)), size
            without = window_attention(q[:, -1:], torch.cat([k[:, :at], k[:, at + 1:]], 1), torch.cat([v[:, :at], v[:, at + 1:]], 1))
            k[:, at] = -each
            # (a key less moves the others to other places of the sums)
            close(window_attention(q[:, -1:], k, v), without, 4 * UNIT[dtype] + 256 * UNIT[torch.float32], "without it")


def test_first_token_of_the_lowest_key(cuda_device):
    """Keys set to a finite lowest value, as padding is masked: a query that sees nothing else gives their values."""
    from isa.kernels.transformer_block import window_attention

    g = torch.Generator(device=cuda_device).manual_seed(3)
    q, k, v = (torch.randn(1, 12, 2, 64, generator=g, device=cuda_device) for _ in range(3))
    k[:, :4] = -1e30
    out = window_attention(q.abs(), k, v)
    assert torch.isfinite(out).all()
    close(out[:, :1], v[:, :1], 4 * UNIT[torch.float32], "the first token")
    plain = torch.softmax((q.abs().double().transpose(1, 2) @ k.double().permute(0, 2, 3, 1).contiguous() * 0.125).masked_fill(
        torch.ones(12, 12, device=cuda_device).triu(1).bool(), -torch.inf), -1) @ v.double().transpose(1, 2)
    close(out[:, 4:], plain.transpose(1, 2)[:, 4:], 64 * UNIT[torch.float32], "past the padding")
