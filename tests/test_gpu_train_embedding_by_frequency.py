"""Ids numbered by frequency, as a vocabulary often is: the frequent ones lie in one range of the sort, beside each other."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_train_embedding import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab, tokens", [(50304, 9000), (50304, 65537), (513, 30000), (140001, 20000), (3, 9000), (129, 5000)])
def test_matches_formulas(cuda_device, vocab, tokens):
    """By lists that a wave kept and by all keys again, with few and with many tokens of a step inside, in ranges of 1 row to 512."""
    for dim in (8, 20):
        print(f"[case] {tokens} of {vocab} x {dim}", flush=True)
        ids, w = make(cuda_device, (tokens,), vocab, dim, torch.float32, seed=dim)
        check(cuda_device, ids, w, padding=1)
        check(cuda_device, ids.sort().values, w)  # whole steps of one row
        check(cuda_device, ids[torch.randperm(tokens, device=cuda_device) % 64], w)  # few rows, again and again


def fastest(call, turns=10):
    times = []
    for _ in range(turns):
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        for _ in range(5):
            call()
        end.record()
        end.synchronize()
        times.append(begin.elapsed_time(end))
    return min(times)


def test_order_of_the_vocabulary_costs_little(cuda_device):
    """65536 tokens: the block with half of them takes some time more, not seven times as much as a step of any order."""
    from isa.kernels.transformer_block import embedding

    ids, w = make(cuda_device, (65536,), 50304, 64, torch.bfloat16)
    other = torch.randperm(50304, device=cuda_device)[ids]
    w.requires_grad_(True)
    dy = torch.randn(65536, 64, device=cuda_device).bfloat16()
    a, b = (fastest(lambda: torch.autograd.grad(embedding(i, w), w, dy)) for i in (ids, other))
    print(f"  by frequency {a * 200:.0f} us a step, in any order {b * 200:.0f}", flush=True)
    assert a <= 4.0 * b
