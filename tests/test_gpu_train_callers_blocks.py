"""GPT around blocks of a caller's own, which know nothing of its seeds."""

from __future__ import annotations

import functools

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from isa.operators.block import GPT, Block, DropoutSeed, WindowAttention
from tests.test_gpu_train_flags import DIM, P, VOCAB, _dropped, run  # noqa: F401  (a fixture)


class Theirs(nn.Module):
    """Attention's and FFN's places, and a module, or whatever else, under the name that Block has its probability by."""

    def __init__(self, dropout):
        super().__init__()
        self.dropout, self.attention, self.fc = dropout, nn.Identity(), nn.Linear(DIM, DIM)

    def forward(self, branch, stream, cache=None):
        if branch is not None:
            stream = stream + branch
        y = self.fc(stream)
        return (self.dropout(y) if callable(self.dropout) else y), stream


class TheirsSeeded(Theirs):
    def forward(self, branch, stream, cache=None, seed=None, site=0):
        self.got = None if seed is None else (seed.tolist(), site)
        return super().forward(branch, stream, cache)


class TheirsAround(nn.Module):
    """Passes on what it gets."""

    def __init__(self, block):
        super().__init__()
        self.block, self.dropout, self.attention = block, block.dropout, nn.Identity()

    def forward(self, *args, **kwargs):
        return self.block(*args, **kwargs)


def make(of_model, *blocks):
    torch.manual_seed(0)
    model = GPT(VOCAB, 20, DIM, nn.ModuleList(blocks), of_model)
    model.seed = DropoutSeed(key=1)
    return model


@pytest.mark.parametrize("theirs", [lambda: nn.Dropout(0.5), lambda: nn.Identity(), lambda: None, lambda: functools.partial(F.dropout, p=0.5),
                                    lambda: 0.5], ids=["Dropout", "Identity", "None", "function", "number"])
def test_blocks_without_seeds(dropped, theirs):  # noqa: F811
    model = make(0.0, Theirs(theirs()), Theirs(theirs()))
    assert run(model, dropped) == [] and model.seed.state.tolist() == [1, 0]
    # with the model's own dropout, and beside blocks that take seeds
    assert run(make(P, Theirs(theirs()), Theirs(theirs())), dropped) == [0, 5]
    ours = Block(DIM, WindowAttention(DIM, 3), nn.Linear(DIM, DIM), P)
    assert run(make(0.0, Theirs(theirs()), ours), dropped) == [3, 4]


def test_blocks_with_seeds_get_theirs(dropped):  # noqa: F811
    model = make(0.0, TheirsSeeded(0.5), TheirsAround(TheirsSeeded(0.5)), Theirs(0.5))
    run(model, dropped)
    assert model.blocks[0].got == ([1, 0], 1) and model.blocks[1].block.got == ([1, 0], 3)
    assert model.seed.state.tolist() == [1, 8]
    model.blocks.eval()
    run(model, dropped)
    assert model.blocks[0].got is None and model.seed.state.tolist() == [1, 8]


@pytest.mark.gpu
def test_blocks_without_seeds_train(cuda_device):
    torch.manual_seed(0)
    model = make(0.0, Theirs(nn.Dropout(0.5)), Theirs(nn.Dropout(0.5))).to(cuda_device)
    ids = torch.randint(0, VOCAB, (2, 7), device=cuda_device)
    model(ids).sum().backward()
    assert all(p.grad is not None for p in model.parameters()) and model.seed.state.tolist() == [1, 0]
    assert not torch.equal(model(ids), model(ids))  # their own dropout
