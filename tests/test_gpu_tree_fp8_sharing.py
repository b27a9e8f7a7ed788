"""packed_tree_attention_fp8 called from several threads and captures: what they share."""
from __future__ import annotations

import threading

import pytest
import torch

import jetspec_b200 as jb

from helpers import bits_equal
from test_gpu_tree_fp8 import DEVICE, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("counts", [[40, 3, 64], [2, 1, 4]])
def test_threads_on_one_stream(counts):
    """Equal shapes, other data: every call gives what it gives alone."""
    prefixes = [900, 4000, 33]
    cases = [Case(prefixes, counts, seed=40 + i) for i in range(2)]
    want = [case.run() for case in cases]
    torch.cuda.synchronize()
    wrong, failed = [0, 0], []

    def work(i):
        try:
            for _ in range(10):
                outs = [cases[i].run() for _ in range(30)]
                wrong[i] += sum(not bits_equal(out, want[i]) for out in outs)
        except BaseException as error:  # reported by the main thread
            failed.append(error)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed and wrong == [0, 0]
    assert jb.read_device_errors() == 0


@pytest.mark.parametrize("counts", [[40, 3, 64], [2, 1, 4]])
def test_graphs_replay_beside_each_other_and_beside_eager_calls(counts):
    """Captured one after the other on one stream, replayed on three at the same time."""
    cases = [Case([9000, 4000, 33], counts, seed=50 + i) for i in range(3)]
    want = [case.run() for case in cases]
    graphs, outs = [], []
    capture = torch.cuda.Stream()
    for case in cases[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=capture):
            outs.append(case.run())
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    with torch.cuda.stream(capture):
        beside = []
        for _ in range(20):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
            beside += [cases[2].run() for _ in range(3)]
    torch.cuda.synchronize()
    assert all(bits_equal(out, want[2]) for out in beside)
    assert bits_equal(outs[0], want[0]) and bits_equal(outs[1], want[1])
    assert jb.read_device_errors() == 0


def test_memory_stays_bounded_over_many_batch_sizes():
    """Every total of packed nodes from 1 to 48: one scratch buffer of the stream, not 48."""
    cases = [Case([64] * n, [1] * n, kv_heads=1, groups=2, dim=16, block=64, seed=n)
             for n in (1, 48)]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        cases[1].run()
        held = torch.cuda.memory_allocated(DEVICE)
        for n in range(1, 48):
            case = Case([64] * n, [1] * n, kv_heads=1, groups=2, dim=16, block=64, seed=n)
            case.run()
            del case
        assert torch.cuda.memory_allocated(DEVICE) - held < 1 << 20
        want = cases[0].run()
    stream.synchronize()
    assert bits_equal(want, cases[0].run())
