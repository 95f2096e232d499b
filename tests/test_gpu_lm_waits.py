"""Bounded waits of the language-model row kernels.

MAG_CUDA_TC_TEST_STALL=1 gives a kernel a first wait that nothing completes, before anything that it would have to
wait for is under way.  The wait runs out, every warp and block leaves, mag_cuda_synchronize returns
MAG_CUDA_E_DEVICE_WAIT once, and the next call on the same device is right."""
import os

import numpy as np
import pytest

import mag_b200 as MB
from gpu_util import device

pytestmark = pytest.mark.gpu


def up(a):
    a = np.ascontiguousarray(a, np.float32)
    t = device().tensor((a.size,))
    t.write(a.reshape(-1))
    return t


def stalled(call, results):
    """call() three times, the second with a wait that runs out: the last gives the first's results."""
    d = device()
    call()
    assert d.L.mag_cuda_synchronize(d.p) == 0
    want = [t.read().view(np.uint32) for t in results]
    os.environ["MAG_CUDA_TC_TEST_STALL"] = "1"
    try:
        call()
        rc = d.L.mag_cuda_synchronize(d.p)
    finally:
        del os.environ["MAG_CUDA_TC_TEST_STALL"]
    assert rc == MB.E_DEVICE_WAIT
    assert d.L.mag_cuda_synchronize(d.p) == 0  # reported once
    for t in results:
        t.write(np.full(t.numel, np.nan, np.float32))
    call()
    assert d.L.mag_cuda_synchronize(d.p) == 0
    for t, w in zip(results, want):
        assert np.array_equal(t.read().view(np.uint32), w)


@pytest.mark.parametrize("rows,cols", [(5, 9000), (200, 16384), (301, 16001), (100, 32768)])
def test_norm_backward_of_wide_rows(rows, cols):
    """Clusters of two and of six blocks, several rows each: no block goes on to its next row."""
    d = device()
    g = np.random.default_rng([0x6E, rows, cols])
    dy, h = (up(g.normal(0, 1, (rows, cols))) for _ in range(2))
    w, rstd, dx, dw = up(g.normal(1, 0.2, cols)), up(np.ones(rows)), up(np.zeros((rows, cols))), up(np.zeros(cols))
    stalled(lambda: d.rmsnorm_rows_backward(rows, cols, dx, dw, dy, h, w, rstd), [dx, dw])


# narrow tiles of 16, 32, 64 and 128 rows of x, K whole and split over clusters; pairs
@pytest.mark.parametrize("block", [True, False])
@pytest.mark.parametrize("m,k,n", [(4, 4096, 256), (4, 300, 1000), (20, 2048, 130), (20, 128, 4096), (60, 4096, 512), (60, 256, 700),
                                   (100, 4096, 600), (100, 200, 2000), (1024, 256, 4096), (1000, 2500, 4000)])
def test_matmul_e4m3(m, k, n, block):
    d = device()
    g = np.random.default_rng([0x6F, m, k, n])

    def operand(rows, blocks):
        q = np.zeros((rows, MB.e4m3_ld(k)), np.uint8)
        q[:, :k] = g.integers(0, 0x7F, (rows, k))
        return up(q.view(np.float32)), up(g.uniform(0.5, 2, (-(-rows // 128) if blocks else rows, MB.e4m3_ld(k) // 128)))

    (xq, xs), (yq, ys), r = operand(m, False), operand(n, block), d.tensor((n, m))
    stalled(lambda: d.matmul_e4m3(m, k, n, r, xq, xs, yq, ys, y_block=block), [r])
