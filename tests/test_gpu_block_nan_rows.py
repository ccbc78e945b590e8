"""A NaN that a query or its keys hold reaches the query's result, whatever kernel takes the call and
however its keys are cut: a diverged model is seen at any length of its cache."""

from __future__ import annotations

import math

import pytest
import torch

from tests.block_helpers import UNIT, attention64, close

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def inputs(dev, b, m, n, h, kv, d, dtype, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [torch.randn(*shape, generator=g, device=dev).to(dtype)
            for shape in ((b, m, h, d), (b, n, kv, d), (b, n, kv, d), (b, m, h, d))]


def tolerance(dtype):  # 16 bits: p and out rounded; fp32: scores of some 10 and sums of d terms
    return 64 * UNIT[dtype] if dtype == torch.float32 else 4 * UNIT[dtype]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("queries", [1, 2, 60])
@pytest.mark.parametrize("keys", [1, 40, 200, 1000])
def test_nan_query(cuda_device, keys, queries, dtype):
    from isa.kernels.transformer_block import window_attention

    print(f"[case] NaN query, {queries} of {keys} keys, {dtype}", flush=True)
    lost = max(0, queries - keys)  # queries that see nothing: zeros, whatever they hold
    q, k, v, _ = inputs(cuda_device, 2, queries, keys, 4, 2, 64, dtype, keys + queries)
    want = attention64(q, k, v, None, 0, 0.125, None)[0]
    q[1, -1, 2, 5] = math.nan
    got = window_attention(q, k, v)
    assert torch.isnan(got[1, -1, 2]).all()
    got[1, -1, 2] = want[1, -1, 2].to(got)
    close(got, want, tolerance(dtype), "the other rows")
    assert torch.count_nonzero(got[:, :lost]) == 0


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("window", [None, 100])
def test_nan_keys_of_ragged_sequences(cuda_device, window, dtype):
    """All keys that a token sees are NaN, in sequences that are cut into few and many pieces."""
    from isa.kernels.transformer_block import window_attention

    lengths = [1, 40, 200, 1000, 0]
    print(f"[case] NaN keys, window {window}, {dtype}", flush=True)
    q, k, v, _ = inputs(cuda_device, 5, 1, 1000, 4, 2, 64, dtype, 1)
    k[:, :, 0] = math.nan
    want = attention64(q, torch.nan_to_num(k), v, window, 0, 0.125, lengths)[0]
    got = window_attention(q, k, v, window=window, key_lengths=torch.tensor(lengths, device=cuda_device))
    assert torch.isnan(got[:4, :, :2]).all() and torch.count_nonzero(got[4]) == 0
    close(got[:, :, 2:], want[:, :, 2:], tolerance(dtype), "the other head")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 30), (1, 1000), (70, 70)], ids=str)
def test_nan_query_in_the_gradients(cuda_device, shape, dtype):
    """Its own gradient and those of the keys that it sees are NaN; other rows' and heads' are not."""
    from isa.kernels.transformer_block import window_attention

    m, n = shape
    print(f"[case] gradients of a NaN query, {shape}, {dtype}", flush=True)
    q, k, v, g = inputs(cuda_device, 2, m, n, 4, 2, 64, dtype, 3)
    q[0, m // 2, 1] = math.nan
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    dq, dk, dv = torch.autograd.grad(window_attention(*leaves), leaves, g)
    assert torch.isnan(dq[0, m // 2, 1]).all()
    rest = torch.ones(dq.shape[:3], dtype=torch.bool, device=cuda_device)
    rest[0, m // 2, 1] = False
    assert torch.isfinite(dq[rest]).all()
    seen = n - m + m // 2 + 1
    for t in (dk, dv):
        assert torch.isnan(t[0, :seen, 0]).all()
        assert torch.isfinite(t[0, :, 1]).all() and torch.isfinite(t[1]).all()
