"""Captured calls of the language-model rows: what happens to their buffers between replays.

A graph's replay runs without the library's bookkeeping of pending clears and asynchronous copies, so a
buffer that a captured call uses is cleared at once, and its copies are ordered with the stream at once."""
import numpy as np
import pytest

import mag_b200 as MB
from gpu_util import device

pytestmark = pytest.mark.gpu

EPS = 1e-6


def up(a):
    a = np.ascontiguousarray(a, np.float32)
    t = device().tensor((a.size,))
    t.write(a.reshape(-1))
    return t


def capture(d, calls):
    """The calls once eagerly, then as a graph of the device's stream; returns what replays it."""
    import torch
    stream = torch.cuda.ExternalStream(d.stream, device=f"cuda:{d.ordinal}")
    for c in calls:
        c()
    d.sync()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=stream, capture_error_mode="thread_local"):
        for c in calls:
            c()

    def replay():
        with torch.cuda.stream(stream):
            gr.replay()
    replay.calls = calls  # whose buffers the graph uses
    return replay


def norm_graph(rows=6, cols=256):
    """A captured norm: its replay, input, result and what an eager call gives for the input."""
    d = device()
    a = np.random.default_rng([0x6A, rows, cols]).normal(0, 1, (rows, cols)).astype(np.float32)
    x, w, y, other = up(a), up(np.ones(cols)), up(np.zeros(rows * cols)), up(np.zeros(rows * cols))
    replay = capture(d, [lambda: d.rmsnorm_rows(rows, cols, x, w, EPS, y=y)])
    d.rmsnorm_rows(rows, cols, x, w, EPS, y=other)
    return d, replay, x, y, other.read()


def test_a_cleared_input_is_zero_in_the_replay():
    d, replay, x, y, _ = norm_graph()
    replay()
    x.fill_zero()
    replay()
    assert not y.read().any()
    assert not x.read().any()


def test_a_cleared_result_holds_the_replay():
    d, replay, x, y, want = norm_graph()
    y.fill_zero()
    replay()
    assert np.array_equal(y.read(), want)
    y.fill_zero()
    assert not y.read().any()
    replay()
    assert np.array_equal(d.op("NEG", y).read(), -want)


def test_a_cleared_part_and_a_later_clear_keep_their_order():
    d, replay, x, y, want = norm_graph()
    replay()
    y.write(np.full(8, 5, np.float32))  # part of the result, by the host
    assert np.array_equal(y.read()[8:], want[8:]) and np.all(y.read()[:8] == 5)
    y.fill_zero()
    replay()
    replay()
    assert np.array_equal(y.read(), want)


def test_a_product_adds_to_what_a_replay_left():
    """MATMUL adds to what its result's storage holds; a clear before the replay does not make that zero."""
    d, replay, x, y, want = norm_graph(4, 4)
    one = np.arange(16, dtype=np.float32)
    a, b = d.from_numpy(np.eye(4, dtype=np.float32), (4, 4)), d.from_numpy(one, (4, 4))
    y.fill_zero()
    replay()
    written = up(want)  # the same contents by the host: what the product makes of them is not this test's concern
    for t in (y, written):
        r = MB.Tensor(d, (4, 4), view_of=t)
        r.t.op = MB.OP["MATMUL"]
        r.t.op_inputs[0], r.t.op_inputs[1] = a.ptr, b.ptr
        r.inputs = [a, b]
        d.exec(r)
    assert not np.array_equal(written.read(), one)
    assert np.array_equal(y.read(), written.read())


def test_a_replay_waits_for_uploads_and_downloads():
    """256 MB by the copy engine take milliseconds, the replay less than one."""
    import torch
    rows, cols = 1 << 16, 1024
    d = device()
    g = np.random.default_rng(0x6B)
    old, new = (np.repeat(g.normal(0, 1, (1, rows)).astype(np.float32), cols, 0).T.copy() for _ in range(2))
    x, w, y = up(old), up(np.ones(cols)), up(np.zeros(rows * cols))
    replay = capture(d, [lambda: d.rmsnorm_rows(rows, cols, x, w, EPS, y=y)])
    first = y.read()
    host = torch.from_numpy(new).pin_memory()
    got = torch.empty(rows * cols).pin_memory()
    d.download_async(y, got.data_ptr(), got.numel() * 4)
    d.upload_async(x, host.data_ptr(), host.numel() * 4)
    replay()
    second = y.read()
    d.copies_sync()
    z = up(np.zeros(rows * cols))
    d.rmsnorm_rows(rows, cols, x, w, EPS, y=z)
    assert np.array_equal(x.read(), new.reshape(-1))
    assert np.array_equal(second, z.read())
    assert np.array_equal(got.numpy(), first)
    # a download of the result alone, then a replay that overwrites it at once
    x.write(old)
    d.download_async(y, got.data_ptr(), got.numel() * 4)
    replay()
    d.copies_sync()
    assert np.array_equal(got.numpy(), second)
    assert np.array_equal(y.read(), first)


def test_a_graph_keeps_its_scratch_when_the_device_grows_its_own():
    """A device of its own, whose scratch is 1 MiB after the small call: the larger one needs 148 parts of 4096
    columns, 2.4 MB, so the scratch moves; what it held is allocated again and overwritten."""
    d = MB.Device()
    try:
        g = np.random.default_rng(0x6C)

        def buffers(rows, cols):
            t = [d.tensor((rows * cols,)) for _ in range(3)] + [d.tensor((cols,)) for _ in range(2)] + [d.tensor((rows,))]
            for b in t:
                b.write(g.normal(1, 0.3, b.numel).astype(np.float32))
            return t  # dx, dy, h, dw, w, rstd

        def backward(rows, cols, t):
            d.rmsnorm_rows_backward(rows, cols, t[0], t[3], t[1], t[2], t[4], t[5])

        small, large = buffers(300, 512), buffers(300, 4096)
        replay = capture(d, [lambda: backward(300, 512, small)])
        want = [small[i].read() for i in (0, 3)]
        backward(300, 4096, large)
        d.sync()
        fill = [d.tensor((1 << 16,)) for _ in range(16)]  # 4 MiB from the pool that took the old scratch back
        for t in fill:
            t.write(np.full(t.numel, np.nan, np.float32))
        for i in (0, 3):
            small[i].write(np.full(small[i].numel, np.nan, np.float32))
        replay()
        d.sync()
        for i, a in zip((0, 3), want):
            assert np.array_equal(small[i].read(), a)
        for t in fill:
            assert np.isnan(t.read()).all()
        del replay, small, large, fill
    finally:
        d.close()
