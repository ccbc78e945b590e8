"""WindowCache on the device: its count on the host holds beside HIP graphs that append to it, and gradients
that would miss what passes through it are refused."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_appends_that_a_graph_records(cuda_device):
    from isa.operators.block import WindowCache

    c = WindowCache(2, 8, 2, 8, device=cuda_device)
    k, v = (torch.randn(2, 2, 2, 8, device=cuda_device) for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.append(k, v)
    torch.cuda.current_stream().wait_stream(side)
    c.lengths.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.append(k, v)
    for i in range(3):
        print(f"[case] replay {i}", flush=True)
        k.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert c.lengths.tolist() == [2 * i + 2] * 2 and c.longest() == 2 * i + 2
        assert torch.equal(c.k[:, 2 * i: 2 * i + 2], k)
    with pytest.raises(RuntimeError, match="do not fit"):
        c.append(torch.cat([k, k], 1), torch.cat([v, v], 1))
    c.append(k, v)
    assert c.lengths.tolist() == [8, 8]
    with pytest.raises(RuntimeError, match="do not fit"):
        c.append(k, v)
    c.lengths.zero_()
    c.append(k, v)
    assert c.lengths.tolist() == [2, 2]


def test_gradients_through_a_cache_are_refused(cuda_device):
    from isa.operators.block import GPT, Block, WindowAttention

    torch.manual_seed(0)
    blocks = torch.nn.ModuleList(Block(32, WindowAttention(32, 2, window=8), torch.nn.Linear(32, 32)) for _ in range(2))
    model = GPT(20, 16, 32, blocks).to(cuda_device)
    ids = torch.randint(0, 20, (2, 6), device=cuda_device)
    whole = model(ids)
    caches = model.caches(2, 8)
    out = model(ids, caches)  # without no_grad: the values are right
    torch.testing.assert_close(out, whole, rtol=1e-4, atol=1e-5)
    with pytest.raises(RuntimeError, match="train without a cache"):
        out.sum().backward()
    with torch.no_grad():
        again = model.caches(2, 8)
        torch.testing.assert_close(model(ids, again), out, rtol=0, atol=0)
    whole.sum().backward()
    assert all(p.grad is not None for p in model.parameters())
    # a frozen projection: nothing passes through the keys, but the first block's output still does
    for block in model.blocks:
        block.attention.qkv.requires_grad_(False)
    with pytest.raises(RuntimeError, match="train without a cache"):
        model(ids, model.caches(2, 8)).sum().backward()
    # nothing that needs a gradient before the caches
    model.requires_grad_(False)
    model.blocks[1].ffn.requires_grad_(True)
    model(ids, model.caches(2, 8)).sum().backward()
    assert model.blocks[1].ffn.weight.grad is not None
