"""A dropout seed that is not where a capture needs it."""

from __future__ import annotations

import pytest
import torch

from isa.operators.block import DropoutSeed


def test_a_seed_does_not_move_while_a_graph_is_recorded(monkeypatch):
    """A recorded copy would read its host memory again in each replay (CPU only: the refusal comes before any copy)."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    s = DropoutSeed(key=5)
    with pytest.raises(RuntimeError, match="before one is captured"):
        s.step(3, torch.device("cuda", 0))
    assert s.state.tolist() == [5, 0] and s.state.device.type == "cpu"
    assert s.step(3, torch.device("cpu")).tolist() == [5, 0]  # where it is, it steps


@pytest.mark.gpu
def test_first_steps_in_a_capture(cuda_device):
    from isa.kernels.transformer_block import dropout

    x = torch.ones(4, 64, device=cuda_device)
    s = DropoutSeed(key=5)
    graph, refused = torch.cuda.CUDAGraph(), []
    print("[case] a seed in host memory", flush=True)
    with torch.cuda.graph(graph):
        try:
            s.step(1, cuda_device)
        except RuntimeError as e:
            refused.append(str(e))
        x.mul_(1.0)
    assert len(refused) == 1 and "before one is captured" in refused[0]
    print("[case] a seed that was moved first", flush=True)
    s.step(1, torch.device("cuda"))
    for device in (cuda_device, torch.device("cuda")):  # one device by either name
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = dropout(x, 0.5, s.step(1, device))
        for _ in range(3):
            before = s.state.clone()
            graph.replay()
            torch.cuda.synchronize()
            assert s.state.tolist() == [5, int(before[1]) + 1]
            assert torch.equal(y, dropout(x, 0.5, before))
