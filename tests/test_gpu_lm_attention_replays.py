"""Attention and cache calls after and beside one another: captured ones share no scratch and no counters, and a read sees the write before it."""
import numpy as np
import pytest

import mag_b200 as MB
from gpu_util import device
from test_gpu_lm_attention import Batch, blank, ints, up
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


@pytest.mark.parametrize("rows,heads,dim", [(1, 1, 16), (40, 8, 128), (3000, 4, 64)])
def test_reads_follow_writes_at_once(rows, heads, dim):
    """Slots written again and again and read after each write, without a wait by the host: every read gives what was last written."""
    d, n = device(), heads * dim
    c = d.kv_cache(rows // 16 + 1, heads, dim, 16)
    g = np.random.default_rng([0x52, rows])
    slot = ints(g.permutation(rows))
    sides = [up(g.normal(0, 1, (rows, n))) for _ in range(3)]
    outs = [blank(rows, n) for _ in range(12)]
    for i in range(0, 12, 2):
        d.kv_write(c, rows, slot, sides[i % 3], sides[(i + 1) % 3])
        d.kv_read(c, rows, slot, k=outs[i], v=outs[i + 1])
    first = []
    for side in sides:  # each alone
        d.kv_write(c, rows, slot, side, side)
        one, two = blank(rows, n), blank(rows, n)
        d.sync()
        d.kv_read(c, rows, slot, k=one, v=two)
        first.append(one.read())
        assert np.array_equal(first[-1], two.read())
    for i, o in enumerate(outs):
        assert np.array_equal(o.read(), first[i % 3]), i
