"""GPT's forward pass alone in a HIP graph, with gradients enabled, beside graphs of its leaves that were made on the
default stream; and its backward pass there, which is refused before it reaches one of them."""

from __future__ import annotations

import pytest
import torch
import torch.nn as nn

from isa.operators import block
from isa.operators.block import Embedding
from tests.test_gpu_train_model import make_gpt

pytestmark = pytest.mark.gpu


def theirs(model):
    model.positions = nn.Embedding.from_pretrained(torch.randn(40, 48), freeze=False)


def own_forward(model):
    table = model.positions
    table.forward = lambda at: nn.functional.embedding(at, table.weight)


def scaled_table(model):
    model.positions = Embedding(40, 48, scale=3.0)


CHANGES = {"as made": lambda model: None, "scaled positions": scaled_table, "a caller's positions": theirs, "a caller's forward": own_forward}


@pytest.fixture(name="ids")
def _ids(cuda_device):
    return torch.randint(0, 70, (3, 11), device=cuda_device)


def warm(model, ids):
    """A step on a side stream before any capture, as torch asks for: libraries load and allocate in their first calls."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(model(ids).sum(), list(model.parameters()))
    torch.cuda.current_stream().wait_stream(side)


def captured(work):
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = work()
    return graph, out


def test_a_backward_pass_finds_that_it_is_captured(cuda_device, ids, monkeypatch):
    """The check runs in the backward pass, before any of the model's nodes. (No graph lives here, and the pass ends at
    the check.)"""
    seen = []

    def check(leaves):
        seen.append((torch.cuda.is_current_stream_capturing(), len(list(leaves))))
        raise RuntimeError("ends here")

    monkeypatch.setattr(block, "leaves_can_be_captured", check)
    model = make_gpt(cuda_device)
    warm(model, ids)

    def work():
        with pytest.raises(RuntimeError, match="ends here"):
            model(ids).sum().backward()
        return ids + 1

    graph, out = captured(work)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ids + 1) and seen == [(True, len(list(model.parameters())))]
    assert all(p.grad is None for p in model.parameters())
    model(ids).sum().backward()  # eager passes have no check
    assert len(seen) == 1


@pytest.mark.parametrize("change", CHANGES.values(), ids=CHANGES)
def test_forward_beside_a_living_graph(cuda_device, ids, change):
    model = make_gpt(cuda_device)
    change(model)
    model.to(cuda_device)
    warm(model, ids)
    params = list(model.parameters())
    living = model(ids)
    print("[case] forward alone", flush=True)
    graph, out = captured(lambda: model(ids))
    for _ in range(3):
        ids.copy_(torch.randint(0, 70, ids.shape, device=cuda_device))
        graph.replay()
        torch.cuda.synchronize()
        want = model(ids)
        assert torch.equal(out, want)
        torch.randn(500, 500, device=cuda_device).sum().item()
    print("[case] an eager backward pass of the recorded result", flush=True)
    graph, out = captured(lambda: model(ids))  # (of ids that are not written since)
    graph.replay()
    want = model(ids)
    up = torch.randn_like(out)
    got = torch.autograd.grad(out, params, up)
    assert all(torch.equal(a, b) for a, b in zip(got, torch.autograd.grad(want, params, up)))
    del living


def test_backward_beside_a_living_graph_is_refused(cuda_device, ids):
    model = make_gpt(cuda_device)
    warm(model, ids)
    living = model(ids)

    def work():
        with pytest.raises(RuntimeError, match="before a step with that leaf is captured"):
            model(ids).sum().backward()
        return ids + 1

    graph, out = captured(work)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ids + 1) and all(p.grad is None for p in model.parameters())
    living.sum().backward()
    assert all(p.grad is not None for p in model.parameters())
