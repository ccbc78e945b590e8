"""Whose flag says whether a model's parts drop: each module's own, as nn.Dropout's in its place would."""

from __future__ import annotations

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from isa.operators import block
from isa.operators.block import GPT, Block, DropoutSeed, WindowAttention
from tests.block_helpers import close
from tests.train_helpers import factors

VOCAB, DIM, P = 30, 48, 0.25


def make(dropout=P, of_blocks=P, layers=2):
    torch.manual_seed(0)
    blocks = nn.ModuleList(Block(DIM, WindowAttention(DIM, 3, window=9, sinks=2), nn.Linear(DIM, DIM), of_blocks) for _ in range(layers))
    return GPT(VOCAB, 20, DIM, blocks, dropout)


class Echo(nn.Module):
    """In an attention's place."""

    def forward(self, x, cache=None):
        return x


@pytest.fixture(name="dropped")
def _dropped(monkeypatch):
    """The sites that drop, in order; the operators' places are taken by torch's functions."""
    sites = []

    def drop(x, p, seed, *, site=0):
        sites.append(site)
        return x

    def norm(x, w, b, eps):
        return F.layer_norm(x, w.shape, w, b, eps)

    monkeypatch.setattr(block, "embedding", lambda ids, w, *, position_weight=None, **_: F.embedding(ids, w))
    monkeypatch.setattr(block, "dropout", drop)
    monkeypatch.setattr(block, "layer_norm", norm)
    monkeypatch.setattr(block, "add_layer_norm", lambda x, r, w, b, eps: (norm(x + r, w, b, eps), x + r))
    monkeypatch.setattr(block, "dropout_add_layer_norm",
                        lambda x, r, w, b, eps, *, p, seed, site: (drop(x, p, seed, site=site), norm(x + r, w, b, eps), x + r)[1:])
    return sites


def run(model, dropped):
    for b in model.blocks:
        b.attention = Echo()
    dropped.clear()
    model(torch.zeros(1, 4, dtype=torch.int64))
    return list(dropped)


def test_each_modules_own_flag(dropped):
    model = make()
    assert run(model, dropped) == [0, 2, 3, 4, 5]
    model.blocks[0].eval()
    assert run(model, dropped) == [0, 3, 4, 5]
    model.train()
    model.blocks[1].eval()  # which takes the first block's output, too
    assert run(model, dropped) == [0, 2, 5]
    model.train().requires_grad_(False)
    for b in model.blocks:
        b.eval()
    assert run(model, dropped) == [0, 5]
    model.eval()
    assert run(model, dropped) == []
    model.blocks[1].train()
    assert run(model, dropped) == [3, 4]


def test_no_numbers_are_drawn_where_none_drop(dropped):
    model = make(dropout=0.0)
    model.seed = DropoutSeed(key=3)
    for b in model.blocks:
        b.eval()
    assert run(model, dropped) == [] and model.seed.state.tolist() == [3, 0]
    model.blocks[1].train()
    assert run(model, dropped) == [3, 4] and model.seed.state.tolist() == [3, 6]
    model = make(of_blocks=0.0)
    model.training = False  # the model's own alone
    assert run(model, dropped) == [] and model.seed is None


@pytest.mark.gpu
@pytest.mark.parametrize("frozen", [0, 1])
def test_a_block_that_evaluates_in_a_model_that_trains(cuda_device, frozen):
    """fp32 in two orders of summation: some 300 roundings of 2^-24 in the logits of two blocks, 500 in the gradients."""
    model = make().to(cuda_device)
    model.seed = DropoutSeed(key=7)
    model.blocks[frozen].eval()
    ids = torch.randint(0, VOCAB, (2, 12), device=cuda_device)
    up = torch.randn(2, 12, VOCAB, device=cuda_device)
    got = model(ids)
    assert model.seed.state.tolist() == [7, 6]

    def drop(site, t):
        if site in ((2,), (3, 4))[frozen]:
            return t
        return t * factors(24, DIM, P, (7, 0), site).float().to(cuda_device).view(t.shape)

    x = drop(0, F.embedding(ids, model.tokens.weight) + model.positions.weight[:12])
    for i, b in enumerate(model.blocks):
        if i:
            x = x + drop(1 + 2 * i, branch)  # noqa: F821
        x = x + drop(2 + 2 * i, b.attention(F.layer_norm(x, (DIM,), b.ln1.weight, b.ln1.bias)))
        branch = b.ffn(F.layer_norm(x, (DIM,), b.ln2.weight, b.ln2.bias))
    x = x + drop(5, branch)
    want = F.linear(F.layer_norm(x, (DIM,), model.ln_f.weight, model.ln_f.bias), model.tokens.weight)
    close(got, want, 300 * 2.0 ** -24, "logits")
    params = list(model.parameters())
    for a, b, (name, _) in zip(torch.autograd.grad(got, params, up), torch.autograd.grad(want, params, up), model.named_parameters()):
        close(a, b, 500 * 2.0 ** -24, name)
