"""WindowCache on the device: its count on the host holds beside HIP graphs that append to it."""

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
