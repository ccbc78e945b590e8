"""One dropout seed under several threads, on several streams, and in a checkpoint: no offset is drawn twice."""

from __future__ import annotations

import copy
import pickle
import threading
import time

import pytest
import torch

from isa.operators.block import DropoutSeed


def test_threads_draw_one_after_the_other():
    """While one thread is between its copy and its addition, others wait."""
    s, drawn, inside = DropoutSeed(key=1), [], []

    class Slow(torch.Tensor):
        def clone(self):
            inside.append(1)
            assert len(inside) == 1
            time.sleep(0.02)
            inside.pop()
            return self.as_subclass(torch.Tensor).clone()

    s.state = s.state.as_subclass(Slow)

    def run():
        for _ in range(3):
            drawn.append(s.step(4, torch.device("cpu")).tolist())

    threads = [threading.Thread(target=run) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert sorted(drawn) == [[1, 4 * i] for i in range(12)] and s.state.tolist() == [1, 48]


def test_copies_and_pickles_go_on_from_their_state():
    s = DropoutSeed(key=9)
    s.step(5, torch.device("cpu"))
    for other in (copy.deepcopy(s), pickle.loads(pickle.dumps(s))):
        assert other.step(2, torch.device("cpu")).tolist() == [9, 5] and other.state.tolist() == [9, 7]
    assert s.state.tolist() == [9, 5]
    # what a checkpoint keeps, and a run that goes on from it
    kept = s.state.clone()
    resumed = DropoutSeed(key=0)
    resumed.state.copy_(kept)
    assert resumed.step(1, torch.device("cpu")).tolist() == [9, 5]


@pytest.mark.gpu
def test_streams_draw_one_after_the_other(cuda_device):
    """Steps on streams in turn, each behind a queue of work that the next one's stream does not have."""
    s = DropoutSeed(key=1)
    s.step(0, cuda_device)
    a = torch.randn(2048, 2048, device=cuda_device)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    drawn = []
    for turn in range(12):
        with torch.cuda.stream(streams[turn % 3]):
            if turn % 3 == 0:
                for _ in range(20):
                    a @ a
            drawn.append(s.step(4, cuda_device))
    torch.cuda.synchronize()
    assert [d.tolist() for d in drawn] == [[1, 4 * i] for i in range(12)] and s.state.tolist() == [1, 48]
    # a copy of a seed that was used, and one that is used in a capture between eager steps
    t = copy.deepcopy(s)
    assert t.step(1, cuda_device).tolist() == [1, 48] and s.state.tolist() == [1, 48]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = s.step(4, cuda_device)
    with torch.cuda.stream(streams[0]):
        assert s.step(4, cuda_device).tolist() == [1, 48]
    torch.cuda.synchronize()
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert got.tolist() == [1, 52 + 4 * i]
