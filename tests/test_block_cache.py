"""WindowCache keeps its sequences within its capacity and GPT within its table of positions, before
anything is launched (an index past the end would end the process on the GPU). On the CPU: the
cache is torch's tensors alone."""

from __future__ import annotations

import pytest
import torch

from isa.operators.block import GPT, WindowCache


def cache(capacity=8, batch=2):
    return WindowCache(batch, capacity, 2, 8, device="cpu")


def tokens(n, batch=2):
    return torch.randn(batch, n, 2, 8), torch.randn(batch, n, 2, 8)


def test_appends_add_up_to_the_capacity():
    c = cache()
    k, v = tokens(8)
    c.append(k[:, :5], v[:, :5])
    with pytest.raises(RuntimeError, match="do not fit"):
        c.append(*tokens(4))
    assert c.lengths.tolist() == [5, 5]  # nothing was written
    c.append(k[:, 5:], v[:, 5:])
    assert torch.equal(c.k, k) and torch.equal(c.v, v) and c.lengths.tolist() == [8, 8]
    with pytest.raises(RuntimeError, match="do not fit"):
        c.append(*tokens(1))
    with pytest.raises(RuntimeError, match="do not fit"):
        cache().append(*tokens(9))


def test_lengths_that_the_caller_sets_count():
    """Sequences of several lengths, and a cache that is used again."""
    c = cache()
    c.append(*tokens(8))
    c.lengths.copy_(torch.tensor([3, 6]))  # a padded prompt's true lengths
    k, v = tokens(2)
    c.append(k, v)
    assert c.lengths.tolist() == [5, 8]
    assert torch.equal(c.k[0, 3:5], k[0]) and torch.equal(c.v[1, 6:8], v[1])
    with pytest.raises(RuntimeError, match="do not fit"):
        c.append(*tokens(1))
    c.lengths.zero_()
    c.append(*tokens(8))
    c.lengths = torch.tensor([7, 1], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="do not fit"):
        c.append(*tokens(2))
    c.append(*tokens(1))
    assert c.lengths.tolist() == [8, 2]


@pytest.mark.parametrize("made_inside", [False, True])
def test_inference_mode(made_inside):
    if made_inside:
        with torch.inference_mode():
            c = cache()
    else:
        c = cache()
    with torch.inference_mode():
        c.append(*tokens(5))
        c.append(*tokens(3))
        with pytest.raises(RuntimeError, match="do not fit"):
            c.append(*tokens(1))
        c.lengths.fill_(2)
        c.append(*tokens(6))
        with pytest.raises(RuntimeError, match="do not fit"):
            c.append(*tokens(1))
        assert c.lengths.tolist() == [8, 8]


def test_sequences_end_with_the_table_of_positions():
    """(blocks that would need a GPU are left out: the refusal comes before them)"""
    model = GPT(20, 6, 16, torch.nn.ModuleList())
    with pytest.raises(RuntimeError, match="table of 6 positions"):
        model(torch.zeros(2, 7, dtype=torch.int64))
    c = cache()
    c.append(*tokens(5))
    with pytest.raises(RuntimeError, match="table of 6 positions"):
        model(torch.zeros(2, 2, dtype=torch.int64), [c])
    with pytest.raises(RuntimeError, match="CUDA"):  # one more fits, and gets to the last norm
        model(torch.zeros(2, 1, dtype=torch.int64), [c])
