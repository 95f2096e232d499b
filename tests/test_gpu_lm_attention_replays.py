"""Captured attention calls whose replays run beside one another: they share no scratch and no counters."""
import numpy as np
import pytest

import mag_b200 as MB
from gpu_util import device
from test_gpu_lm_attention import Batch
from test_gpu_lm_graphs import capture

pytestmark = pytest.mark.gpu


def graph_of(d, call):
    """The call as a graph of the device's stream, once eagerly before."""
    import torch
    stream = torch.cuda.ExternalStream(d.stream, device=f"cuda:{d.ordinal}")
    call()
    d.sync()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=stream, capture_error_mode="thread_local"):
        call()
    return gr


@pytest.mark.parametrize("seqs", [[(1, 9000)], [(1, 700), (1, 1900), (1, 40)], [(1, 900 + 7 * i) for i in range(60)], [(1, 2500), (40, 300)]])
def test_replays_on_streams_of_their_own(seqs):
    """Sequences that several blocks share, so that the last block of each joins their parts; two graphs and eager calls beside
    them."""
    import torch
    d = device()
    batches = [Batch(seqs, 8, 2, 64, 16, key=k) for k in (1, 2, 3)]
    want = [b.run() for b in batches]
    graphs = [graph_of(d, b.call) for b in batches[:2]]
    streams = [torch.cuda.Stream() for _ in graphs]
    for b in batches:
        for t in (b.out, b.lse):
            t.write(np.full(t.numel, np.nan, np.float32))
    d.sync()
    for _ in range(30):
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        batches[2].call()
    torch.cuda.synchronize()
    for b, w in zip(batches, want):
        got = b.results()
        assert all(np.array_equal(x.view(np.uint32), y.view(np.uint32)) for x, y in zip(got, w))
    del graphs


def test_a_replay_of_two_calls():
    """Two calls of one graph have counters each."""
    d = device()
    batches = [Batch([(1, 5000), (1, 30)], 8, 2, 64, 16, key=k) for k in (1, 2)]
    want = [b.run() for b in batches]
    replay = capture(d, [b.call for b in batches])
    for _ in range(3):
        for b in batches:
            for t in (b.out, b.lse):
                t.write(np.full(t.numel, np.nan, np.float32))
        replay()
        for b, w in zip(batches, want):
            assert all(np.array_equal(x.view(np.uint32), y.view(np.uint32)) for x, y in zip(b.results(), w))


def test_more_graphs_than_the_device_keeps_counters_for():
    """The first 512 captured graphs have counters that the device keeps; those of later ones lie in their scratch."""
    import test_gpu_lm_attention as T
    d = MB.Device()
    old, T.device = T.device, lambda: d
    try:
        batches = [Batch([(1, 3000), (1, 30)], 8, 2, 64, 16, key=k) for k in (1, 2)]
        want = [b.run() for b in batches]
        graphs = [graph_of(d, batches[i % 2].call) for i in range(516)]
        import torch
        stream = torch.cuda.ExternalStream(d.stream, device=f"cuda:{d.ordinal}")
        for i in (0, 1, 511, 512, 513, 515, 514):
            b, w = batches[i % 2], want[i % 2]
            for t in (b.out, b.lse):
                t.write(np.full(t.numel, np.nan, np.float32))
            for _ in range(2):
                with torch.cuda.stream(stream):
                    graphs[i].replay()
            assert all(np.array_equal(x.view(np.uint32), y.view(np.uint32)) for x, y in zip(b.results(), w)), i
        del graphs
    finally:
        T.device = old
