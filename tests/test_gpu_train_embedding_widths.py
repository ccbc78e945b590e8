"""The tables' gradients at every number of lanes and pieces that a row's width leads to, by tiles and by rows alone, with
rows longer than a tile. Tolerances as in test_gpu_train_embedding."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_train_embedding import check, make

pytestmark = pytest.mark.gpu


# 16-byte pieces of a row: 8, 16, 32 and 64 lanes with one each, 64 with two, three and four, and rows of several such steps
@pytest.mark.parametrize("pieces", [2, 8, 9, 16, 17, 25, 32, 33, 64, 65, 128, 129, 192, 193, 256, 300])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_widths(cuda_device, pieces, dtype):
    n = 16 // dtype.itemsize
    for tokens in ((4, 1025), (3, 333)):
        for dim in (n * pieces, n * pieces - n // 2 - 1):
            print(f"[case] {tokens} tokens of {dim} columns, {dtype}", flush=True)
            ids, w = make(cuda_device, tokens, 300, dim, dtype, seed=pieces)
            p = torch.randn(50, dim, device=cuda_device).to(dtype)
            at = torch.randint(0, 50, tokens, device=cuda_device)
            check(cuda_device, ids, w, 0.5, at, p, padding=7)
