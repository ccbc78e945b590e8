"""GPT's tables as their modules are: a caller's scale, padding and hooks on either of them, as when each is called."""

from __future__ import annotations

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.nn.modules.module import register_module_forward_hook

from isa.operators import block
from isa.operators.block import GPT, Embedding
from tests.block_helpers import UNIT, close

VOCAB, PLACES, DIM = 30, 12, 16


def stand_in(ids, weight, *, scale=1.0, positions=None, position_weight=None, padding_index=None):
    """The operator's definition, on any device."""
    y = scale * F.embedding(ids, weight, padding_idx=padding_index)
    if position_weight is not None:
        at = torch.arange(ids.shape[-1], device=ids.device) if positions is None else positions
        y = y + F.embedding(at, position_weight)
    return y


def scaled(model):
    model.positions = Embedding(PLACES, DIM, scale=5.0)


def padded(model):
    model.positions = Embedding(PLACES, DIM, padding_idx=2)
    nn.init.normal_(model.positions.weight)


def scaled_and_padded_tokens(model):
    model.tokens = Embedding(VOCAB, DIM, padding_idx=3, scale=0.5)


def hooked(table):
    def change(model):
        getattr(model, table).register_forward_hook(lambda module, args, out: 3.0 * out)
    return change


def pre_hooked(table):
    def change(model):
        getattr(model, table).register_forward_pre_hook(lambda module, args: (args[0].clamp(max=4), *args[1:]))
    return change


def backward_hooked(table):
    def change(model):
        getattr(model, table).register_full_backward_pre_hook(lambda module, grads: tuple(2.0 * g for g in grads))
    return change


def own_forward(table):
    def change(model):
        module = getattr(model, table)
        module.forward = lambda ids: -F.embedding(ids, module.weight)
    return change


CHANGES = {"as made": lambda model: None, "scaled positions": scaled, "padded positions": padded,
           "scaled and padded tokens": scaled_and_padded_tokens,
           **{f"{f.__name__} {table}": f(table) for table in ("tokens", "positions")
              for f in (hooked, pre_hooked, backward_hooked, own_forward)}}


def both_called(model, ids, at):
    """What a call of each module gives."""
    at = torch.arange(ids.shape[1], device=ids.device) if at is None else at
    return model.tokens(ids) + model.positions(at)


def check(dev, change, tol):
    torch.manual_seed(0)
    model = GPT(VOCAB, PLACES, DIM, nn.ModuleList())
    change(model)
    model.to(dev)
    ids = torch.randint(0, VOCAB, (3, 9), device=dev)
    ids[0, :4] = 3
    up = torch.randn(3, 9, DIM, device=dev)
    tables = [model.tokens.weight, model.positions.weight]
    for at in (None, torch.randint(0, PLACES, (3, 9), device=dev)):
        if at is not None:
            at[1, :5] = 2
        got, want = model._embed(ids, at), both_called(model, ids, at)
        close(got, want, tol, "y")
        for a, b in zip(torch.autograd.grad(got, tables, up), torch.autograd.grad(want, tables, up)):
            close(a, b, 40 * UNIT[torch.float32], "gradient")  # fp32 sums of at most 27 terms, in two orders


@pytest.mark.parametrize("change", CHANGES.values(), ids=CHANGES)
def test_tables_are_what_their_modules_say(monkeypatch, change):
    monkeypatch.setattr(block, "embedding", stand_in)
    check(torch.device("cpu"), change, 2 * UNIT[torch.float32])


def test_hooks_of_all_modules_see_both_tables(monkeypatch):
    monkeypatch.setattr(block, "embedding", stand_in)
    model, seen = GPT(VOCAB, PLACES, DIM, nn.ModuleList()), []
    handle = register_module_forward_hook(lambda module, args, out: seen.append(module))
    try:
        model._embed(torch.zeros(1, 3, dtype=torch.int64), None)
    finally:
        handle.remove()
    assert seen == [model.tokens, model.positions]


def test_both_tables_are_one_call_where_nothing_speaks_against_it(monkeypatch):
    calls = []
    monkeypatch.setattr(block, "embedding", lambda *args, **how: calls.append(how) or stand_in(*args, **how))
    model = GPT(VOCAB, PLACES, DIM, nn.ModuleList())
    model._embed(torch.zeros(1, 3, dtype=torch.int64), None)
    assert len(calls) == 1 and calls[0]["position_weight"] is model.positions.weight


@pytest.mark.gpu
@pytest.mark.parametrize("change", CHANGES.values(), ids=CHANGES)
def test_tables_on_the_operator(cuda_device, change):
    """(the sum of two rounded rows against one rounding: three roundings of numbers no larger than some 5 times y's norm)"""
    check(cuda_device, change, 16 * UNIT[torch.float32])


@pytest.mark.gpu
def test_a_scaled_position_table_against_torch(cuda_device):
    """fp32 in two orders of summation: some 100 roundings of 2^-24 in the logits, as many again in the gradients."""
    torch.manual_seed(0)
    model = GPT(VOCAB, PLACES, DIM, nn.ModuleList())
    model.positions = Embedding(PLACES, DIM, padding_idx=2, scale=5.0)
    nn.init.normal_(model.positions.weight)
    model.to(cuda_device)
    ids = torch.randint(0, VOCAB, (3, 9), device=cuda_device)
    up = torch.randn(3, 9, VOCAB, device=cuda_device)
    w, p = model.tokens.weight, model.positions.weight
    x = F.embedding(ids, w) + 5.0 * F.embedding(torch.arange(9, device=cuda_device), p, padding_idx=2)
    want = F.linear(F.layer_norm(x, (DIM,), model.ln_f.weight, model.ln_f.bias), w)
    got = model(ids)
    close(got, want, 100 * UNIT[torch.float32], "logits")
    grads = [torch.autograd.grad(y, (w, p), up) for y in (got, want)]
    close(grads[0][0], grads[1][0], 200 * UNIT[torch.float32], "tokens")
    close(grads[0][1], grads[1][1], 200 * UNIT[torch.float32], "positions")
    assert torch.count_nonzero(grads[0][1][2]) == 0
