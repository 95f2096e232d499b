"""Language-model row operators on the GPU against plain implementations in 64 bits.

u = 2^-24 is half an f32 step relative to the value; every tolerance below is a count of such
roundings.  e4m3 rounding is off by at most half a step: 2^-4 of the value, or 2^-10 below 2^-6."""
import ctypes as C
import math

import numpy as np
import pytest

import mag_b200 as MB
from gpu_util import device

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-6
VALUES = MB.e4m3_values().astype(np.float64)


def rng(*key):
    return np.random.default_rng([0x1A, *key])


def up(a):
    """A row-major array on the device."""
    a = np.ascontiguousarray(a, np.float32)
    t = device().tensor((max(1, a.size),))
    if a.size:
        t.write(a.reshape(-1))
    return t


def out(*shape):
    """A result buffer full of NaN bits, so that values left unwritten show."""
    n = max(1, int(np.prod(shape)))
    t = device().tensor((n,))
    t.write(np.full(n, np.nan, np.float32))
    return t


def get(t, *shape):
    return t.read()[:int(np.prod(shape))].reshape(shape)


def get_bytes(t, rows, ld):
    return t.read().view(np.uint8)[:rows * ld].reshape(rows, ld)


def half_step(v):
    """Half a step of e4m3 at magnitude v."""
    _, e = np.frexp(np.minimum(np.abs(v), 448.0))
    return 2.0 ** (np.maximum(e - 4, -9) - 1)


def operand(rows, cols, block, seed, spread=0.5):
    """Bytes, scales and values of a random e4m3 operand."""
    g = rng(seed, rows, cols, block)
    ld, n = MB.e4m3_ld(cols), -(-rows // 128) if block else rows
    q = np.zeros((rows, ld), np.uint8)
    b = g.integers(0, 256, (rows, cols)).astype(np.uint8)
    b[(b & 0x7F) == 0x7F] = 0
    q[:, :cols] = b
    s = np.exp(g.normal(0, spread, (n, ld // 128))).astype(np.float32) * 0.01
    full = np.repeat(s, 128, 0)[:rows] if block else s
    return q, s, VALUES[q] * np.repeat(full.astype(np.float64), 128, 1)


def check_quantized(q, s, v, block, rel):
    """q, s against the 64-bit values v (rows x cols), each known within rel of the kernel's own."""
    rows, cols = v.shape
    ld, n = MB.e4m3_ld(cols), -(-rows // 128) if block else rows
    assert q.shape == (rows, ld) and s.shape == (n, ld // 128)
    assert not q[:, cols:].any()
    p = np.zeros((n * 128 if block else rows, ld))
    p[:rows, :cols] = v
    top = np.abs(p.reshape(n, 128 if block else 1, ld // 128, 128)).max((1, 3))
    want = np.maximum(top, 2.0 ** -100) / 448.0
    assert np.all(np.abs(s - want) <= want * (rel + 2 * U))  # the maximum's own error, the division
    each = np.repeat(np.repeat(s.astype(np.float64), 128, 0)[:rows] if block else s.astype(np.float64), 128, 1)[:, :cols]
    t = v / each
    # q is formed from v (448 / amax): the value's error, the factor's and the product's rounding and that of
    # s here, then half a step of the result (at the larger magnitude where rounding crosses a power of two)
    slack = np.abs(t) * (rel + 3 * U)
    assert np.all(np.abs(VALUES[q[:, :cols]] - t) <= half_step(np.abs(t) + slack) + slack)


# ------------------------------------------------------------------ quantiser
SIZES = [(1, 1), (1, 128), (3, 100), (128, 128), (129, 127), (130, 257), (257, 1000), (64, 4096), (1000, 4), (1, 5001)]


@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("block", [False, True])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_quantize(rows, cols, block, transpose):
    d = device()
    x = (rng(rows, cols).normal(0, 1, (rows, cols)) * np.exp(rng(1, rows).normal(0, 3, (rows, 1)))).astype(np.float32)
    a, b = (cols, rows) if transpose else (rows, cols)
    q, s = d.e4m3(a, b, block)
    q.write(np.full(q.numel, np.nan, np.float32))
    d.quantize_e4m3(rows, cols, up(x), q, s, block=block, transpose=transpose)
    v = (x.T if transpose else x).astype(np.float64)
    n = -(-a // 128) if block else a
    check_quantized(get_bytes(q, a, MB.e4m3_ld(b)), get(s, n, MB.e4m3_ld(b) // 128), v, block, 0.0)


def test_quantize_special_groups():
    d = device()
    x = np.zeros((6, 256), np.float32)
    x[0, 3] = 2.0 ** -120          # below the floor: zeros
    x[1, :128] = 3.0e38            # the largest magnitudes
    x[2, 5], x[2, 6] = np.nan, 1.0
    x[3, 7], x[3, 8] = np.inf, -2.0
    x[4, 130] = -1.0
    x[5, :] = np.float32(1e-40)    # subnormal inputs
    q, s = d.e4m3(6, 256)
    d.quantize_e4m3(6, 256, up(x), q, s)
    b, sc = get_bytes(q, 6, 256), get(s, 6, 2)
    tiny = np.float32(2.0 ** -100) / np.float32(448)
    assert not (b[0] & 0x7F).any() and np.all(sc[0] == tiny)
    assert np.all(b[1, :128] == 0x7E) and sc[1, 1] == tiny
    assert np.all((b[2, :128] & 0x7F) == 0x7F) and np.isnan(sc[2, 0]) and sc[2, 1] == tiny
    assert (b[3, 7] & 0x7F) == 0x7F and not (b[3, 8] & 0x7F).any() and np.isinf(sc[3, 0])
    assert b[4, 130] == 0xFE and sc[4, 1] == np.float32(1) / np.float32(448)
    assert not (b[5] & 0x7F).any() and np.all(sc[5] == tiny)


# -------------------------------------------------------------------- product
def product_bound(x, y, groups):
    """|x||y|^T times the roundings on an output's way: in a group of 128, four instructions of 32
    products each lose at most one f32 unit (2 u) per product and per accumulation of the absolute
    sum; then each of the groups' sums is scaled (2 u) and added (u)."""
    return (np.abs(x) @ np.abs(y).T) * (2 * U * (32 + 4) + U * (groups + 3))


PRODUCTS = [(1, 128, 8), (1, 100, 7), (1, 4096, 300), (2, 1, 1), (3, 129, 130), (4, 4096, 1024), (8, 512, 129), (9, 300, 257),
            (16, 1024, 384), (17, 640, 100), (31, 256, 1000), (33, 2000, 65), (64, 128, 512), (100, 1500, 700),
            (127, 384, 127), (128, 256, 128), (129, 1000, 513), (200, 4100, 260), (256, 512, 256), (257, 640, 1025),
            (520, 1300, 771), (1030, 256, 40), (2100, 300, 2001), (5000, 128, 1030), (700, 1664, 5000), (300, 4096, 9000), (260, 256, 33000),
            (48, 14336, 700), (64, 700, 20000), (40, 5000, 1300)]


@pytest.mark.parametrize("block", [True, False])
@pytest.mark.parametrize("m,k,n", PRODUCTS)
def test_matmul_e4m3(m, k, n, block):
    d = device()
    xq, xs, x = operand(m, k, False, 2)
    yq, ys, y = operand(n, k, block, 3)
    r = out(m, n)
    args = (up(xq.view(np.float32)), up(xs), up(yq.view(np.float32)), up(ys))
    d.matmul_e4m3(m, k, n, r, *args, y_block=block)
    got = get(r, m, n)
    want = x @ y.T
    assert np.all(np.abs(got - want) <= product_bound(x, y, xs.shape[1]))
    d.matmul_e4m3(m, k, n, r, *args, y_block=block)
    assert np.array_equal(get(r, m, n).view(np.uint32), got.view(np.uint32))  # the same sums every time


def test_matmul_writes_nothing_else():
    d = device()
    m, k, n = 37, 300, 51
    xq, xs, x = operand(m, k, False, 4)
    yq, ys, y = operand(n, k, True, 5)
    r = d.tensor((m * n + 64,))
    r.write(np.full(m * n + 64, 7.5, np.float32))
    keep = [up(xq.view(np.float32)), up(xs), up(yq.view(np.float32)), up(ys)]
    d.matmul_e4m3(m, k, n, r.data_ptr + 128, *keep)  # 32 values in
    a = r.read()
    assert np.all(a[:32] == 7.5) and np.all(a[32 + m * n:] == 7.5)
    assert np.all(np.abs(a[32:32 + m * n].reshape(m, n) - x @ y.T) <= product_bound(x, y, 3))
    d.matmul_e4m3(m, k, n, r.data_ptr + 4, *keep)  # a result that is only 4-byte aligned
    assert np.array_equal(r.read()[1:1 + m * n], a[32:32 + m * n])


@pytest.mark.parametrize("m", [3, 40, 300])
def test_matmul_nan_stays_in_its_rows(m):
    d = device()
    k, n = 384, 200
    xq, xs, x = operand(m, k, False, 6)
    yq, ys, y = operand(n, k, False, 7)
    xq[1, 200] = 0x7F
    ys[5, 1] = np.inf
    r = out(m, n)
    d.matmul_e4m3(m, k, n, r, up(xq.view(np.float32)), up(xs), up(yq.view(np.float32)), up(ys), y_block=False)
    got = get(r, m, n)
    assert np.isnan(got[1]).all() and not np.isfinite(got[:, 5]).any()
    ok = np.ones((m, n), bool)
    ok[1] = False
    ok[:, 5] = False
    assert np.isfinite(got[ok]).all()


def test_matmul_subnormal_and_exact_values():
    """Small whole numbers with scale 1: every sum is exact in f32, so are the results."""
    d = device()
    for m, k, n in ((2, 512, 64), (20, 512, 96), (140, 512, 300)):
        g = rng(8, m)
        codes = np.array([0x00, 0x38, 0x40, 0x44, 0xB8, 0xC0, 0x01, 0x81], np.uint8)  # 0, 1, 2, 3, -1, -2, +-2^-9
        xq, yq = codes[g.integers(0, 8, (m, k))], codes[g.integers(0, 8, (n, k))]
        one = lambda a: np.ones((a, k // 128), np.float32)  # noqa: E731
        r = out(m, n)
        d.matmul_e4m3(m, k, n, r, up(xq.view(np.float32)), up(one(m)), up(yq.view(np.float32)), up(one(n)), y_block=False)
        x, y = VALUES[xq], VALUES[yq]
        # products are multiples of 2^-18 up to 9: a sum of 512 of them needs 2^13 * 2^18 at most, so only
        # the bits below 2^-24 of a sum's magnitude (a few hundred) can be lost
        assert np.all(np.abs(get(r, m, n) - x @ y.T) <= product_bound(x, y, 4))
        xq[(xq == 1) | (xq == 0x81)] = 0
        d.matmul_e4m3(m, k, n, r, up(xq.view(np.float32)), up(one(m)), up(yq.view(np.float32)), up(one(n)), y_block=False)
        whole = VALUES[xq] @ np.where(np.abs(y) < 1, 0, y).T
        if not ((yq == 1) | (yq == 0x81)).any():
            assert np.array_equal(get(r, m, n), whole)


# ----------------------------------------------------------------------- norm
NORMS = [(1, 1), (1, 128), (3, 100), (5, 129), (2, 4096), (7, 5000), (1, 8192), (3, 8200), (2, 20000), (1, 40001), (300, 256), (1500, 64),
         (640, 1024)]


def norm_rel(cols):
    """Relative error of v = t rstd w: the sum of squares takes at most cols / 128 additions on a thread
    and 12 in the joins (and the squares' rounding, the mean's division, eps); the root halves it and
    rsqrt adds 2 units; then the sum x + residual and two products."""
    n = cols / 128 + 12 + 4
    return (n / 2 + 4 + 4) * U


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,cols", NORMS + [(400, 13000), (600, 12801), (2, 16385), (300, 20000), (2, 65536), (3, 70001)])
def test_rmsnorm(rows, cols, residual):
    d = device()
    g = rng(9, rows, cols)
    x = g.normal(0, 1, (rows, cols)).astype(np.float32)
    res = (g.normal(0, 2, (rows, cols)) * np.exp(g.normal(0, 1, cols))).astype(np.float32)
    w = g.normal(1, 0.3, cols).astype(np.float32)
    y, h, rstd = out(rows, cols), out(rows, cols), out(rows)
    q, s = d.e4m3(rows, cols)
    q.write(np.full(q.numel, np.nan, np.float32))
    d.rmsnorm_rows(rows, cols, up(x), up(w), EPS, residual=up(res) if residual else None, y=y, q=q, q_scale=s, h=h, rstd=rstd)
    t32 = x + res if residual else x
    assert np.array_equal(get(h, rows, cols), t32)
    t = t32.astype(np.float64)
    root = 1.0 / np.sqrt((t * t).mean(1, keepdims=True) + EPS)
    v = t * root * w
    rel = norm_rel(cols)
    assert np.all(np.abs(get(rstd, rows, 1) - root) <= root * rel)
    assert np.all(np.abs(get(y, rows, cols) - v) <= np.abs(v) * rel)
    check_quantized(get_bytes(q, rows, MB.e4m3_ld(cols)), get(s, rows, MB.e4m3_ld(cols) // 128), v, False, rel)
    # each output alone is the same
    y2, q2, s2 = out(rows, cols), *d.e4m3(rows, cols)
    d.rmsnorm_rows(rows, cols, up(x), up(w), EPS, residual=up(res) if residual else None, y=y2)
    d.rmsnorm_rows(rows, cols, up(x), up(w), EPS, residual=up(res) if residual else None, q=q2, q_scale=s2)
    assert np.array_equal(y2.read(), y.read())
    assert np.array_equal(q2.read().view(np.uint32), q.read().view(np.uint32)) and np.array_equal(s2.read(), s.read())


@pytest.mark.parametrize("rows,cols", [(4, 512), (3, 1001), (2, 30000)])
def test_rmsnorm_in_place_and_unaligned(rows, cols):
    d = device()
    g = rng(10, rows, cols)
    x, res, w = (g.normal(0, 1, sh).astype(np.float32) for sh in ((rows, cols), (rows, cols), cols))
    y, h = out(rows, cols), out(rows, cols)
    d.rmsnorm_rows(rows, cols, up(x), up(w), EPS, residual=up(res), y=y, h=h)
    want_y, want_h = y.read(), h.read()
    bx, br = up(x), up(res)
    d.rmsnorm_rows(rows, cols, bx, up(w), EPS, residual=br, y=bx, h=br)  # the residual stream in place
    assert np.array_equal(bx.read(), want_y) and np.array_equal(br.read(), want_h)
    bx, br = up(x), up(res)
    d.rmsnorm_rows(rows, cols, bx, up(w), EPS, residual=br, y=br, h=bx)
    assert np.array_equal(br.read(), want_y) and np.array_equal(bx.read(), want_h)
    pad = lambda a: np.concatenate([[0.0], a.reshape(-1)])  # noqa: E731
    px, pr, pw, py, ph = up(pad(x)), up(pad(res)), up(pad(w)), out(rows * cols + 2), out(rows * cols + 2)
    d.rmsnorm_rows(rows, cols, px.data_ptr + 4, pw.data_ptr + 4, EPS, residual=pr.data_ptr + 4, y=py.data_ptr + 4,
                   h=ph.data_ptr + 4)
    # a thread adds other columns of an unaligned row: both results are within norm_rel of the formula
    assert np.all(np.abs(py.read()[1:-1] - want_y) <= 2 * norm_rel(cols) * np.abs(want_y))
    assert np.array_equal(ph.read()[1:-1], want_h)
    assert np.isnan(py.read()[[0, -1]]).all()


def test_rmsnorm_zero_and_nonfinite_rows():
    d = device()
    cols = 700
    x = np.ones((5, cols), np.float32)
    x[1] = 0.0
    x[2, 3] = np.nan
    x[3, 4] = np.inf
    y, q, s = out(5, cols), *d.e4m3(5, cols)
    d.rmsnorm_rows(5, cols, up(x), up(np.ones(cols)), 0.5, y=y, q=q, q_scale=s)
    a, sc = get(y, 5, cols), get(s, 5, 6)
    assert np.all(a[1] == 0) and np.all(sc[1] == np.float32(2.0 ** -100) / np.float32(448))
    assert np.isnan(a[2]).all() and np.isnan(sc[2]).all()
    assert np.isnan(a[3, 4]) and np.all(np.delete(a[3], 4) == 0)  # 1 / sqrt(inf) = 0
    assert np.all(np.abs(a[[0, 4]] - 1 / math.sqrt(1.5)) <= norm_rel(cols))


@pytest.mark.parametrize("rows,cols", NORMS + [(5000, 96), (33, 8192), (200, 9001), (300, 20000), (2, 65536), (3, 70001)])
def test_rmsnorm_backward(rows, cols):
    d = device()
    g = rng(11, rows, cols)
    h = (g.normal(0, 1, (rows, cols)) * np.exp(g.normal(0, 1, cols))).astype(np.float32)
    dy, dh = (g.normal(0, 1, (rows, cols)).astype(np.float32) for _ in range(2))
    w = g.normal(1, 0.3, cols).astype(np.float32)
    h64, dy64, w64 = (a.astype(np.float64) for a in (h, dy, w))
    rstd = (1.0 / np.sqrt((h64 * h64).mean(1) + EPS)).astype(np.float32)
    r = rstd[:, None].astype(np.float64)
    u = dy64 * w64
    along = (u * h64).mean(1, keepdims=True)
    # mean(u h): two products' roundings and the additions, of the absolute sum
    n = cols / 128 + 12 + 4
    err_along = np.abs(u * h64).mean(1, keepdims=True) * n * U
    want = r * (u - h64 * r * r * along)
    tol = 8 * U * r * (np.abs(u) + np.abs(h64 * r * r * along)) + r * np.abs(h64) * r * r * err_along
    dw = (dy64 * h64 * r).sum(0)
    tol_w = (np.abs(dy64 * h64) * r).sum(0) * (rows + 4) * U
    for with_dh in (False, True):
        dx, dwt = out(rows, cols), out(cols)
        d.rmsnorm_rows_backward(rows, cols, dx, dwt, up(dy), up(h), up(w), up(rstd), dh=up(dh) if with_dh else None)
        full = want + dh if with_dh else want
        assert np.all(np.abs(get(dx, rows, cols) - full) <= tol + (U * np.abs(full) if with_dh else 0))
        assert np.all(np.abs(get(dwt, cols) - dw) <= tol_w)
        again = out(cols)
        d.rmsnorm_rows_backward(rows, cols, out(rows, cols), again, up(dy), up(h), up(w), up(rstd))
        assert np.array_equal(again.read(), dwt.read())
    for at in range(3):  # in place, and without dw
        bufs = [up(dy), up(h), up(dh)]
        d.rmsnorm_rows_backward(rows, cols, bufs[at], None, bufs[0], bufs[1], up(w), up(rstd), dh=bufs[2])
        assert np.array_equal(get(bufs[at], rows, cols), get(dx, rows, cols))
        bufs = [up(dy), up(h), up(dh)]
        d.rmsnorm_rows_backward(rows, cols, bufs[at], again, bufs[0], bufs[1], up(w), up(rstd), dh=bufs[2])
        assert np.array_equal(get(bufs[at], rows, cols), get(dx, rows, cols)) and np.array_equal(again.read(), dwt.read())


def test_rmsnorm_backward_no_rows():
    dw = out(40)
    t = out(1)
    device().rmsnorm_rows_backward(0, 40, t, dw, t, t, t, t)
    assert np.all(get(dw, 40) == 0)


def test_rmsnorm_gradient_against_differences():
    d = device()
    rows, cols, e = 3, 300, 1e-5
    g = rng(12)
    x, w, k = g.normal(0, 1, (rows, cols)), g.normal(1, 0.3, cols), g.normal(0, 1, (rows, cols))
    x, w = x.astype(np.float32).astype(np.float64), w.astype(np.float32).astype(np.float64)
    loss = lambda x, w: (x / np.sqrt((x * x).mean(1, keepdims=True) + EPS) * w * k.astype(np.float32)).sum()  # noqa: E731
    y, h, rstd, dx, dw = out(rows, cols), out(rows, cols), out(rows), out(rows, cols), out(cols)
    d.rmsnorm_rows(rows, cols, up(x), up(w), EPS, y=y, h=h, rstd=rstd)
    d.rmsnorm_rows_backward(rows, cols, dx, dw, up(k), h, up(w), rstd)
    vx, vw = g.normal(0, 1, x.shape), g.normal(0, 1, w.shape)
    diff = (loss(x + e * vx, w) - loss(x - e * vx, w)) / (2 * e)
    scale = np.abs(get(dx, rows, cols) * vx).sum()
    assert abs((get(dx, rows, cols) * vx).sum() - diff) <= 1e-5 * scale  # f32 values, e^2 of the difference
    diff = (loss(x, w + e * vw) - loss(x, w - e * vw)) / (2 * e)
    assert abs((get(dw, cols) * vw).sum() - diff) <= 1e-5 * np.abs(get(dw, cols) * vw).sum()


# ------------------------------------------------------------------ log probabilities
def logprobs64(x):
    """lse, entropy and E|x - max| per row, in 64 bits; an empty row as the header says."""
    x = x.astype(np.float64)
    m = x.max(1, keepdims=True)
    with np.errstate(invalid="ignore"):
        dd = np.where(np.isneginf(x), -np.inf, x - np.where(np.isneginf(m), 0, m))
        e = np.exp(dd)
        s = e.sum(1, keepdims=True)
        t = np.where(e > 0, e * np.where(np.isneginf(dd), 0, dd), 0).sum(1, keepdims=True)
    empty = np.isneginf(m[:, 0])
    s1 = np.where(empty[:, None], 1.0, s)
    lse = np.where(empty, -np.inf, np.where(empty, 0, m[:, 0]) + np.log(s1[:, 0]))
    ent = np.where(empty, 0.0, np.log(s1[:, 0]) - (t / s1)[:, 0])
    return lse, ent, (-t / s1)[:, 0]


def best(x, k):
    """The k first columns of each row by (value, lower column)."""
    key = np.where(np.isnan(x), np.inf, x)
    nan_first = np.lexsort((np.broadcast_to(np.arange(x.shape[1]), x.shape), -key, ~np.isnan(x)), axis=1)
    return nan_first[:, :k]


def run_logprobs(x, ids, k, stride=None, what=("logp", "lse", "entropy", "top_logp", "top_id")):
    d = device()
    rows, cols = x.shape
    stride = stride or cols
    buf = np.full((rows, stride), 1e30, np.float32)  # padding that must not be read
    buf[:, :cols] = x
    o = {"logp": out(rows), "lse": out(rows), "entropy": out(rows), "top_logp": out(rows, k), "top_id": out(rows, k)}
    args = {n: o[n] for n in what}
    d.token_logprobs(rows, cols, up(buf), d.ids(ids), top=k, x_stride=stride, **args)
    got = {n: get(o[n], rows, k) if n.startswith("top") else get(o[n], rows) for n in what}
    if "top_id" in got:
        got["top_id"] = got["top_id"].view(np.int32)
    return got


def lp_tol(x, adds):
    """Errors of lse (absolute) and entropy: every term exp(d) is within (|d| + 4) 2u of itself (the rounding
    of d and of its product with log2 e, the exponential's 2 units), the sum has at most `adds` additions,
    its logarithm is within 2 units; the entropy's sum of e d has the same errors weighted by |d|."""
    lse, ent, ed = logprobs64(x)
    rel = 2 * U * (ed + 4) + U * adds
    log = rel + 4 * U * np.abs(np.where(np.isfinite(lse), lse, 0)) + 2 * U * math.log(x.shape[1] + 1)
    x64 = x.astype(np.float64)
    with np.errstate(invalid="ignore"):
        p = np.exp(x64 - np.where(np.isfinite(lse), lse, 0)[:, None])
        dd = np.where(p > 0, np.abs(x64 - x64.max(1, keepdims=True)), 0)
        second = (np.where(p > 0, p * dd * (dd + 6), 0)).sum(1)
    return log, log + ed * rel + 2 * U * second + U * adds * ed


LOGITS = [(1, 1, 1), (1, 5, 5), (4, 32, 32), (3, 33, 7), (2, 1000, 20), (5, 1023, 1), (3, 4097, 32), (300, 256, 4), (700, 1030, 0),
          (5, 50001, 20), (1, 131072, 32), (9, 131072, 5), (2, 262147, 10), (160, 20000, 8), (1, 1000003, 32),
          (148, 66001, 3), (200, 5000, 20), (594, 65537, 2), (1200, 9000, 4)]


@pytest.mark.parametrize("rows,cols,k", LOGITS)
def test_logprobs(rows, cols, k):
    g = rng(13, rows, cols)
    x = g.normal(0, 2.5, (rows, cols)).astype(np.float32)
    hot = g.integers(0, cols, rows)
    x[np.arange(rows), hot] += 8
    ids = np.where(g.random(rows) < 0.5, hot, g.integers(0, cols, rows)).astype(np.int32)
    for stride in (cols, cols + 3):
        got = run_logprobs(x, ids, k, stride)
        lse, ent, _ = logprobs64(x)
        tol, tol_h = lp_tol(x, cols / 128 + 20)
        assert np.all(np.abs(got["lse"] - lse) <= tol)
        xi = x[np.arange(rows), ids].astype(np.float64)
        assert np.all(np.abs(got["logp"] - (xi - lse)) <= tol + U * (np.abs(xi) + np.abs(xi - lse)))
        assert np.all(np.abs(got["entropy"] - ent) <= tol_h)
        want = best(x, k)
        assert np.array_equal(got["top_id"], want)
        v = np.take_along_axis(x, want, 1).astype(np.float64)
        assert np.all(np.abs(got["top_logp"] - (v - lse[:, None])) <= tol[:, None] + U * (np.abs(v) + np.abs(v - lse[:, None])))
    for name in ("logp", "lse", "entropy", "top_logp", "top_id") if k else ("logp", "lse", "entropy"):
        alone = run_logprobs(x, ids, k, None, (name,))
        both = run_logprobs(x, ids, k)
        assert np.array_equal(alone[name], both[name])


@pytest.mark.parametrize("cols", [200, 6000, 70001])
def test_logprobs_masked_rows(cols):
    g = rng(14, cols)
    x = g.normal(0, 2, (8, cols)).astype(np.float32)
    x[0] = -np.inf                                    # nothing left
    x[1, :] = -np.inf
    x[1, cols - 1] = 3.0                              # one left
    x[2, ::2] = -np.inf
    x[3] = np.finfo(np.float32).min                   # the type's lowest value everywhere
    x[4, 5:] = np.finfo(np.float32).min
    x[5, 10:] = -np.inf
    x[6] = 0.0
    x[7, :cols // 2] = -np.inf
    ids = np.array([3, cols - 1, 1, 0, 2, 11, 7, cols - 1], np.int32)
    k = 12
    got = run_logprobs(x, ids, k)
    lse, ent, _ = logprobs64(x)
    tol, tol_h = lp_tol(x, cols / 128 + 20)
    fin = np.isfinite(lse)
    assert np.isneginf(got["lse"][0]) and np.isneginf(got["logp"][0]) and got["entropy"][0] == 0
    assert np.isneginf(got["top_logp"][0]).all()
    assert np.isneginf(got["logp"][5]) and got["logp"][1] == 0 and got["entropy"][1] == 0
    assert np.all(np.abs(got["lse"][fin] - lse[fin]) <= tol[fin])
    # f32 rows at the lowest value: lse = lowest + ln(n) rounds to the lowest, logp = -ln(n) needs the difference
    assert np.all(np.abs(got["entropy"] - ent)[fin] <= tol_h[fin] + 1e-30)
    assert np.array_equal(got["top_id"], best(x, k))


def test_logprobs_ties_and_signed_zeros():
    for cols in (100, 9000, 40000):
        x = np.zeros((4, cols), np.float32)
        x[0, ::2] = -0.0
        x[1] = np.arange(cols) // 7
        x[2] = -(np.arange(cols) // 5)
        x[3, [3, cols - 1, cols // 2]] = 1.0
        got = run_logprobs(x, np.zeros(4, np.int32), 32)
        assert np.array_equal(got["top_id"], best(x, 32))


@pytest.mark.parametrize("order", ["rising", "falling", "few values", "spikes late", "mostly masked"])
def test_logprobs_top_of_awkward_rows(order):
    """Rows that keep beating the bound, or tie with it, everywhere in the row."""
    cols, k = 150003, 32
    g = rng(21)
    x = g.normal(0, 1, (3, cols)).astype(np.float32)
    if order in ("rising", "falling"):
        x = np.sort(x, axis=1)[:, ::1 if order == "rising" else -1]
    elif order == "few values":
        x = np.floor(x * 2)
    elif order == "spikes late":
        x[:, -2000:] += 10
    else:
        x[:] = -np.inf
        x[0, [7, 90000, 140001]] = 1.0
        x[1, 149000:149010] = 2.0
        x[2, ::7] = -1.0
    x = np.ascontiguousarray(np.repeat(x, 60, 0))  # one block a row as well as a cluster a row
    for rows in (3 * 60, 3):
        part = x[:: 180 // rows]
        got = run_logprobs(part, np.zeros(rows, np.int32), k)
        assert np.array_equal(got["top_id"], best(part, k))


def test_logprobs_nan_inf_and_odd_ids():
    cols = 5000
    x = rng(15).normal(0, 1, (5, cols)).astype(np.float32)
    x[1, 77] = np.nan
    x[2, 40] = np.inf
    x[4, [9, 3000]] = np.nan
    got = run_logprobs(x, np.array([-1, 5, 5, cols, 2], np.int32), 3)
    assert got["logp"][0] == 0 and np.isnan(got["logp"][1:]).all()
    assert np.isnan(got["lse"][[1, 2, 4]]).all() and np.isnan(got["entropy"][[1, 2, 4]]).all()
    assert np.isnan(got["top_logp"][[1, 2, 4]]).all()
    assert np.array_equal(got["top_id"], best(x, 3)) and got["top_id"][1, 0] == 77 and got["top_id"][2, 0] == 40


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 5), (2, 1000), (5, 4097), (1, 131072), (300, 257), (3, 50001)])
def test_logprobs_backward(rows, cols):
    d = device()
    g = rng(16, rows, cols)
    x = g.normal(0, 2.5, (rows, cols)).astype(np.float32)
    if cols > 2:
        x[0, ::3] = -np.inf
    ids = g.integers(0, cols, rows).astype(np.int32)
    if rows > 2:
        ids[1] = -1
        x[2] = -np.inf
    lse, ent, _ = logprobs64(x)
    lse32, ent32 = lse.astype(np.float32), ent.astype(np.float32)
    gl, gh = (g.normal(0, 1, rows).astype(np.float32) for _ in range(2))
    live = np.where(ids >= 0, gl, 0)[:, None].astype(np.float64)
    hot = np.zeros((rows, cols))
    hot[np.arange(rows)[ids >= 0], ids[ids >= 0]] = 1
    empty = np.isneginf(lse)[:, None]
    l64 = np.where(empty, 0, lse32.astype(np.float64)[:, None])
    dd = np.where(np.isneginf(x), 0, x - l64)
    p = np.where(np.isneginf(x), 0, np.exp(dd))
    h64 = ent32.astype(np.float64)[:, None]
    for use_l, use_h in ((True, True), (True, False), (False, True)):
        a = live * use_l
        b = gh[:, None].astype(np.float64) * use_h
        want = np.where(empty, 0, a * (hot - p) - b * p * (dd + h64))
        mag = np.abs(a) + np.abs(b) * (np.abs(dd) + np.abs(h64))
        tol = p * mag * (2 * np.abs(dd) + 16) * U + 4 * U * np.abs(a) * hot + 1e-37 * (1 + mag)
        for xs, dxs in ((cols, cols), (cols + 5, cols + 2)):
            bx = np.full((rows, xs), 9.0, np.float32)
            bx[:, :cols] = x
            dx = out(rows, dxs)
            d.token_logprobs_backward(rows, cols, dx, up(bx), d.ids(ids), up(lse32), up(ent32) if use_h else None,
                                      up(gl) if use_l else None, up(gh) if use_h else None, x_stride=xs, dx_stride=dxs)
            got = get(dx, rows, dxs)
            assert np.all(np.abs(got[:, :cols] - want) <= tol)
            assert np.isnan(got[:, cols:]).all()
    t = up(x)
    d.token_logprobs_backward(rows, cols, t, t, d.ids(ids), up(lse32), None, up(gl), None)  # in place
    d.token_logprobs_backward(rows, cols, dx, up(x), d.ids(ids), up(lse32), None, up(gl), None)
    assert np.array_equal(get(t, rows, cols), get(dx, rows, cols))


def test_logprobs_backward_bad_id_is_nan():
    d = device()
    x, dx = up(np.zeros((2, 10))), out(2, 10)
    d.token_logprobs_backward(2, 10, dx, x, d.ids([10, 3]), up(np.full(2, math.log(10))), None, up(np.ones(2)), None)
    got = get(dx, 2, 10)
    assert np.isnan(got[0]).all() and np.isfinite(got[1]).all()


def test_logprobs_gradient_against_differences():
    d = device()
    rows, cols, e = 3, 400, 1e-5
    g = rng(17)
    x = g.normal(0, 2, (rows, cols)).astype(np.float32).astype(np.float64)
    ids = g.integers(0, cols, rows).astype(np.int32)
    gl, gh = (g.normal(0, 1, rows).astype(np.float32).astype(np.float64) for _ in range(2))

    def loss(x):
        lse = np.log(np.exp(x).sum(1))
        lp = x - lse[:, None]
        return (gl * lp[np.arange(rows), ids]).sum() - (gh * (np.exp(lp) * lp).sum(1)).sum()

    lse, ent, dx = out(rows), out(rows), out(rows, cols)
    t = up(x)
    d.token_logprobs(rows, cols, t, lse=lse, entropy=ent)
    d.token_logprobs_backward(rows, cols, dx, t, d.ids(ids), lse, ent, up(gl), up(gh))
    v = g.normal(0, 1, x.shape)
    diff = (loss(x + e * v) - loss(x - e * v)) / (2 * e)
    got = get(dx, rows, cols) * v
    assert abs(got.sum() - diff) <= 1e-5 * np.abs(got).sum()


# ------------------------------------------------------------- offsets past 32 bits
def test_offsets_past_32_bits():
    """Matrices of more than 2^32 bytes (and 2^31 values): their last rows are right."""
    import torch
    d = device()
    g = torch.Generator(device="cuda").manual_seed(5)
    dev = f"cuda:{d.ordinal}"
    last = 3
    # log probabilities: three rows 1.5 * 10^9 logits apart
    cols, stride = 5000, 1_500_000_000
    x = torch.empty(3 * stride, device=dev)
    rows = torch.randn(3, cols, device=dev, generator=g)
    for i in range(3):
        x[i * stride:i * stride + cols] = rows[i]
    ids = torch.tensor([1, 2, cols - 1], dtype=torch.int32, device=dev)
    lse, logp, one = (torch.ones(3, device=dev) for _ in range(3))
    torch.cuda.synchronize()
    d.token_logprobs(3, cols, x.data_ptr(), ids.data_ptr(), logp=logp.data_ptr(), lse=lse.data_ptr(), x_stride=stride)
    d.token_logprobs_backward(3, cols, x.data_ptr(), x.data_ptr(), ids.data_ptr(), lse.data_ptr(), None, one.data_ptr(),
                              x_stride=stride, dx_stride=stride)
    d.sync()
    r64 = rows.double()
    want = r64 - torch.logsumexp(r64, 1, keepdim=True)
    assert torch.all((logp - want.gather(1, ids[:, None].long())[:, 0]).abs() <= 1e-5)
    grad = -want.exp()
    grad[torch.arange(3), ids.long()] += 1
    for i in range(3):
        assert torch.all((x[i * stride:i * stride + cols] - grad[i]).abs() <= 1e-5)
    del x
    # norm and quantiser: 2.2 * 10^9 values
    n, c = 550_000, 4000
    x = torch.randn(n, c, device=dev, generator=g)
    w = torch.ones(c, device=dev)
    q = torch.empty(n, MB.e4m3_ld(c), dtype=torch.uint8, device=dev)
    s = torch.empty(n, MB.e4m3_ld(c) // 128, device=dev)
    tail = x[-last:].double()
    torch.cuda.synchronize()
    d.rmsnorm_rows(n, c, x.data_ptr(), w.data_ptr(), EPS, y=x.data_ptr(), q=q.data_ptr(), q_scale=s.data_ptr())
    d.sync()
    v = (tail / (tail.square().mean(1, keepdim=True) + EPS).sqrt()).cpu().numpy()
    assert np.all(np.abs(x[-last:].cpu().numpy() - v) <= np.abs(v) * norm_rel(c))
    check_quantized(q[-last:].cpu().numpy(), s[-last:].cpu().numpy(), v, False, norm_rel(c))
    q.zero_()
    tail = x[-last:].cpu().numpy().astype(np.float64)
    torch.cuda.synchronize()
    d.quantize_e4m3(n, c, x.data_ptr(), q.data_ptr(), s.data_ptr())
    d.sync()
    check_quantized(q[-last:].cpu().numpy(), s[-last:].cpu().numpy(), tail, False, 0.0)
    qt = torch.empty(c, MB.e4m3_ld(n), dtype=torch.uint8, device=dev)
    st = torch.empty(c, MB.e4m3_ld(n) // 128, device=dev)
    end = n // 128 * 128 - 256
    col = x[end:, -last:].cpu().numpy().astype(np.float64).T
    torch.cuda.synchronize()
    d.quantize_e4m3(n, c, x.data_ptr(), qt.data_ptr(), st.data_ptr(), transpose=True)
    d.sync()
    check_quantized(qt[-last:, end:].cpu().numpy(), st[-last:, end // 128:].cpu().numpy(), col, False, 0.0)
    del x, q, qt
    # product: 70000 x 40000 results, by pairs, and 20 x 120 million by narrow tiles
    for m, n in ((70_000, 40_000), (20, 120_000_000)):
        xq, xs, xv = operand(last, 128, False, 30)
        yq, ys, yv = operand(last, 128, False, 31)
        bx, by = (torch.zeros(k, 128, dtype=torch.uint8, device=dev) for k in (m, n))
        sx, sy = (torch.ones(k, 1, device=dev) for k in (m, n))
        bx[-last:], by[-last:] = torch.from_numpy(xq).to(dev), torch.from_numpy(yq).to(dev)
        sx[-last:], sy[-last:] = torch.from_numpy(xs).to(dev), torch.from_numpy(ys).to(dev)
        r = torch.empty(m, n, device=dev)
        torch.cuda.synchronize()
        d.matmul_e4m3(m, 128, n, r.data_ptr(), bx.data_ptr(), sx.data_ptr(), by.data_ptr(), sy.data_ptr(), y_block=False)
        d.sync()
        assert np.all(np.abs(r[-last:, -last:].cpu().numpy() - xv @ yv.T) <= product_bound(xv, yv, 1))
        assert not r[-last:, 1000:2000].any() and not r[:m - last, -last:].any()  # the rows of zeros
        del bx, by, sx, sy, r
    torch.cuda.empty_cache()


# ---------------------------------------------------------------- as they are used
def test_layer_and_loss_together():
    """One 8-bit layer with its norm, the loss on its logits, and both gradients of the layer."""
    d = device()
    rows, k, n = 150, 520, 1100
    g = rng(18)
    x, res = (g.normal(0, 1, (rows, k)).astype(np.float32) for _ in range(2))
    w = g.normal(1, 0.2, k).astype(np.float32)
    mat = (g.normal(0, 1, (k, n)) / math.sqrt(k)).astype(np.float32)  # the framework's [K][N]
    ids = g.integers(0, n, rows).astype(np.int32)
    gl = np.full(rows, -1.0 / rows, np.float32)
    # forward: norm -> e4m3, weight -> e4m3 (transposed blocks), product, log probabilities
    y, h, rstd = out(rows, k), out(rows, k), out(rows)
    q, qs = d.e4m3(rows, k)
    wq, ws = d.e4m3(n, k, True)
    tw = up(mat)
    d.rmsnorm_rows(rows, k, up(x), up(w), EPS, residual=up(res), y=y, q=q, q_scale=qs, h=h, rstd=rstd)
    d.quantize_e4m3(k, n, tw, wq, ws, block=True, transpose=True)
    logits, logp, lse = out(rows, n), out(rows), out(rows)
    d.matmul_e4m3(rows, k, n, logits, q, qs, wq, ws)
    d.token_logprobs(rows, n, logits, d.ids(ids), logp=logp, lse=lse)
    # backward: logits' gradient, its e4m3 in both orders, dX = dY W^T and dW = X^T dY, the norm's gradient
    dl, dy_, dw_, dx, dg = out(rows, n), out(rows, k), out(k, n), out(rows, k), out(k)
    d.token_logprobs_backward(rows, n, dl, logits, d.ids(ids), lse, None, up(gl), None)
    a, as_ = d.e4m3(rows, n)
    d.quantize_e4m3(rows, n, dl, a, as_)
    b, bs = d.e4m3(k, n, True)
    d.quantize_e4m3(k, n, tw, b, bs, block=True)
    d.matmul_e4m3(rows, n, k, dy_, a, as_, b, bs)
    yt, yts = d.e4m3(k, rows)
    lt, lts = d.e4m3(n, rows)
    d.quantize_e4m3(rows, k, y, yt, yts, transpose=True)
    d.quantize_e4m3(rows, n, dl, lt, lts, transpose=True)
    d.matmul_e4m3(k, rows, n, dw_, yt, yts, lt, lts, y_block=False)
    d.rmsnorm_rows_backward(rows, k, dx, dg, dy_, h, up(w), rstd)

    # each product against 64 bits of unquantised operands: both are off by half a step, 2^-4 of a value
    # or 2^-10 of its scale (of the group's largest magnitude / 448)
    two = (1 + 2.0 ** -4) ** 2 - 1

    def near(got, p, q_):
        floor = 2.0 ** -10 / 448
        pa, qa = np.abs(p), np.abs(q_)
        tol = two * (pa @ qa) + floor * 1.07 * ((pa.max() + 0 * pa) @ qa + pa @ (qa.max() + 0 * qa))
        return np.all(np.abs(got - p @ q_) <= tol)

    t = x.astype(np.float64) + res
    v = t / np.sqrt((t * t).mean(1, keepdims=True) + EPS) * w
    assert near(get(logits, rows, n), v, mat.astype(np.float64))
    z = get(logits, rows, n).astype(np.float64)
    l64 = np.log(np.exp(z).sum(1))
    assert np.all(np.abs(get(logp, rows) - (z[np.arange(rows), ids] - l64)) <= 1e-5)
    p = np.exp(z - l64[:, None])
    p[np.arange(rows), ids] -= 1
    p /= rows
    assert np.all(np.abs(get(dl, rows, n) - p) <= 1e-5 / rows)
    assert near(get(dy_, rows, k), p, mat.T.astype(np.float64))
    assert near(get(dw_, k, n), v.T, p)
    u = get(dy_, rows, k).astype(np.float64)
    r = 1 / np.sqrt((t * t).mean(1, keepdims=True) + EPS)
    want = r * (u * w - t * r * r * (u * w * t).mean(1, keepdims=True))
    assert np.abs(get(dx, rows, k) - want).max() <= 1e-5 * np.abs(want).max()
    assert np.abs(get(dg, k) - (u * t * r).sum(0)).max() <= 1e-5 * np.abs(u * t * r).sum(0).max()


def graph_calls(rows=40, k=384, n=600):
    """The calls of one small step, as closures over buffers that were written once."""
    d = device()
    g = rng(19)
    x, w = up(g.normal(0, 1, (rows, k))), up(g.normal(1, 0.2, k))
    y, h, rstd, dx, dw = out(rows, k), out(rows, k), out(rows), out(rows, k), out(k)
    q, qs = d.e4m3(rows, k)
    wq, ws = d.e4m3(n, k, True)
    mat = up(g.normal(0, 0.05, (k, n)))
    logits, logp, lse, ent, dl, tl, ti = out(rows, n), out(rows), out(rows), out(rows), out(rows, n), out(rows, 5), out(rows, 5)
    ids, gl = d.ids(g.integers(0, n, rows)), up(g.normal(0, 1, rows))
    calls = [
        lambda: d.quantize_e4m3(k, n, mat, wq, ws, block=True, transpose=True),
        lambda: d.rmsnorm_rows(rows, k, x, w, EPS, y=y, q=q, q_scale=qs, h=h, rstd=rstd),
        lambda: d.matmul_e4m3(rows, k, n, logits, q, qs, wq, ws),
        lambda: d.token_logprobs(rows, n, logits, ids, logp=logp, lse=lse, entropy=ent, top=5, top_logp=tl, top_id=ti),
        lambda: d.token_logprobs_backward(rows, n, dl, logits, ids, lse, ent, gl, gl),
        lambda: d.rmsnorm_rows_backward(rows, k, dx, dw, y, h, w, rstd),
    ]
    return calls, x, [logits, logp, lse, ent, tl, ti, dl, dx, dw, y], (rows, k)


@pytest.mark.parametrize("size", [(40, 384, 600), (6, 17000, 300)])
def test_captured_and_replayed(size):
    """Two graphs of the same calls over their own buffers, replayed in turn on new inputs: equal to
    eager calls bit for bit, also after the device's scratch has been grown by other work."""
    import torch
    d = device()
    stream = torch.cuda.ExternalStream(d.stream, device=f"cuda:{d.ordinal}")
    sets = [graph_calls(*size) for _ in range(2)]
    graphs = []
    for calls, _, _, _ in sets:
        for c in calls:
            c()
        d.sync()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=stream, capture_error_mode="thread_local"):
            for c in calls:
                c()
        graphs.append(gr)
    big = 3 << 20
    grown = d.op("SUM", up(np.ones(big)))  # other work on the device's scratch
    assert grown.read()[0] == big
    for turn in range(2):
        fresh = [rng(20, turn, i).normal(0, 1, s[3]).astype(np.float32) for i, s in enumerate(sets)]
        for s, f in zip(sets, fresh):
            s[1].write(f.reshape(-1))
        with torch.cuda.stream(stream):
            for _ in range(2):
                for gr in graphs:
                    gr.replay()
        d.sync()
        got = [[t.read() for t in s[2]] for s in sets]
        for s, g_ in zip(sets, got):
            for c in s[0]:
                c()
            for t, was in zip(s[2], g_):
                assert np.array_equal(t.read().view(np.uint32), was.view(np.uint32))
    del graphs


def test_capture_refuses_unwritten_storage():
    import torch
    d = device()
    stream = torch.cuda.ExternalStream(d.stream, device=f"cuda:{d.ordinal}")
    fresh, x = d.tensor((256,)), up(np.ones(256))
    w, y = up(np.ones(64)), out(256)
    d.rmsnorm_rows(4, 64, x, w, EPS, y=y)
    d.sync()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=stream, capture_error_mode="thread_local"):
        with pytest.raises(MB.CudaError):
            d.rmsnorm_rows(4, 64, fresh, w, EPS, y=y)
        with pytest.raises(MB.CudaError):
            d.rmsnorm_rows(4, 64, x, w, EPS, y=fresh)
        d.rmsnorm_rows(4, 64, x, w, EPS, y=y)
    with torch.cuda.stream(stream):
        gr.replay()
    d.sync()
    assert np.all(np.abs(y.read() - 1 / math.sqrt(1 + EPS)) <= norm_rel(64))
    assert np.all(fresh.read() == 0)


def test_reads_fresh_storage_as_zero():
    """New storage is zero by contract, also where the clear is still pending."""
    d = device()
    y = out(4, 64)
    d.rmsnorm_rows(4, 64, d.tensor((64, 4)), up(np.ones(64)), EPS, y=y)
    assert np.all(y.read() == 0)


def test_calls_are_counted():
    d = device()
    before = d.launches()
    for c in graph_calls()[0]:
        c()
    assert d.launches() >= before + 6
