"""The bytes of e4m3 operands and the bits of their products on the GPU, compared for equality.

A group's scale is s = f32(a f32(1 / 448)) and a byte is the e4m3 value nearest to the quotient v / s as f32
rounds it, ties to even.  Both operations and roundings are IEEE's, so numpy gives the same bits."""
import numpy as np
import pytest

import mag_b200 as MB
from gpu_util import device

pytestmark = pytest.mark.gpu

VALUES = MB.e4m3_values()
TINY = np.float32(2.0 ** -100)


def up(a):
    a = np.ascontiguousarray(a, np.float32)
    t = device().tensor((a.size,))
    t.write(a.reshape(-1))
    return t


def filled(t, byte=0xA5):
    """t with every byte the same, so that bytes left unwritten show."""
    t.write(np.full(t.numel * 4, byte, np.uint8).view(np.float32))
    return t


def get_bytes(t, rows, ld):
    return t.read().view(np.uint8)[:rows * ld].reshape(rows, ld)


def to_e4m3(t):
    """f32 values as e4m3 bytes: steps of 2^-9 below 2^-6, else 3 bits after the leading one; ties to even."""
    t64 = t.astype(np.float64)
    mag = np.minimum(np.abs(np.where(np.isnan(t64), 0, t64)), 448.0)
    _, e = np.frexp(mag)
    step = 2.0 ** np.maximum(e - 4, -9)
    code = np.searchsorted(VALUES[:0x7F].astype(np.float64), np.rint(mag / step) * step).astype(np.uint8)
    code = np.where(np.isnan(t64), 0x7F, np.minimum(code, 0x7E)).astype(np.uint8)
    return np.where(np.isnan(t64), code, code | (np.signbit(t64).astype(np.uint8) << 7))


def quantized(v, block):
    """Bytes [rows][ld] and scales of the f32 matrix v; a NaN in a group makes the whole group NaN."""
    rows, cols = v.shape
    ld, n = MB.e4m3_ld(cols), -(-rows // 128) if block else rows
    p = np.zeros((n * 128 if block else rows, ld), np.float32)
    p[:rows, :cols] = v
    with np.errstate(all="ignore"):
        top = np.abs(p.reshape(n, 128 if block else 1, ld // 128, 128)).max((1, 3))
        s = np.maximum(top, TINY) * (np.float32(1) / np.float32(448))
        each = np.repeat(np.repeat(s, 128, 0)[:rows] if block else s, 128, 1)
        q = to_e4m3(p[:rows] / each)
    q[:, cols:] = 0
    return q, s


def same_bytes(got, want):
    """Equal, NaN of either sign being one value."""
    g, w = (np.where((a & 0x7F) == 0x7F, 0x7F, a) for a in (got, want))
    return np.array_equal(g, w)


def near_ties(rows, seed):
    """Rows of groups whose other values lie at and next to the midpoints of neighbouring e4m3 values."""
    g = np.random.default_rng([0xE4, seed])
    top = np.exp(g.normal(0, 8, rows)).astype(np.float32)
    s = top * (np.float32(1) / np.float32(448))
    mid = (VALUES[:0x7E].astype(np.float64) + VALUES[1:0x7F]) / 2
    v = (mid[None, :] * s[:, None].astype(np.float64)).astype(np.float32)
    v = (v.view(np.int32) + g.integers(-2, 3, v.shape)).astype(np.int32).view(np.float32)
    v *= np.where(g.random(v.shape) < 0.5, -1, 1).astype(np.float32)
    return np.concatenate([top[:, None], v, np.zeros((rows, 1), np.float32)], 1)  # 128 columns


@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("block", [False, True])
@pytest.mark.parametrize("shape", ["ties", "ragged", (2500, 4100), (1, 128), (300, 1001)])
def test_quantized_bytes(shape, block, transpose):
    """Every byte and every scale, at 4-byte aligned addresses too."""
    d = device()
    if shape == "ties":
        v = near_ties(1280, 1)
        if block:  # one largest magnitude for the whole block
            v = v / v[:, :1] * np.repeat(v[::128, :1], 128, 0)
    elif shape == "ragged":
        v = near_ties(257, 2)[:, :101]
    else:
        g = np.random.default_rng([0xE5, *shape])
        v = (g.normal(0, 1, shape) * np.exp(g.normal(0, 1, (shape[0], 1)))).astype(np.float32)
    want, ws = quantized(v, block)
    x = np.ascontiguousarray(v.T if transpose else v)
    for shift in (0, 1):
        q, s = d.e4m3(*v.shape, block)
        filled(q)
        d.quantize_e4m3(*x.shape, up(np.concatenate([np.zeros(shift), x.reshape(-1)])).data_ptr + 4 * shift, q, s, block=block,
                        transpose=transpose)
        assert np.array_equal(s.read().view(np.uint32), ws.reshape(-1).view(np.uint32))
        assert same_bytes(get_bytes(q, v.shape[0], want.shape[1]), want)


@pytest.mark.parametrize("rows,cols", [(300, 4096), (41, 1001), (3, 20000), (2, 70001)])
def test_norm_quantizes_its_own_result(rows, cols):
    """The norm's e4m3 result is that of its f32 result."""
    d = device()
    g = np.random.default_rng([0xE8, rows])
    x, w = g.normal(0, 1, (rows, cols)), g.normal(1, 0.3, cols)
    y, (q, s) = d.tensor((rows * cols,)), d.e4m3(rows, cols)
    filled(q)
    d.rmsnorm_rows(rows, cols, up(x), up(w), 1e-6, y=y, q=q, q_scale=s)
    want, ws = quantized(y.read().reshape(rows, cols), False)
    assert np.array_equal(s.read().view(np.uint32), ws.reshape(-1).view(np.uint32))
    assert same_bytes(get_bytes(q, rows, want.shape[1]), want)


@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("block", [False, True])
@pytest.mark.parametrize("rows,cols", [(7, 300), (7, 301), (140, 141), (130, 17)])
def test_padding_of_groups_with_nan_and_inf(rows, cols, block, transpose):
    """Bytes past the columns are zero whatever the group holds; its own bytes and scales are the rule's."""
    d = device()
    v = np.random.default_rng([0xE6, rows, cols]).normal(0, 1, (rows, cols)).astype(np.float32)
    v[1, cols - 1] = np.nan
    v[3, cols - 2] = np.inf
    v[rows - 1, 0] = -np.inf
    v[5] = 0
    want, ws = quantized(v, block)
    x = np.ascontiguousarray(v.T if transpose else v)
    q, s = d.e4m3(rows, cols, block)
    filled(q)
    d.quantize_e4m3(*x.shape, up(x), q, s, block=block, transpose=transpose)
    got = get_bytes(q, rows, want.shape[1])
    assert not got[:, cols:].any()
    assert same_bytes(got, want)
    assert np.array_equal(s.read(), ws.reshape(-1), equal_nan=True)


@pytest.mark.parametrize("cols", [300, 301, 9001, 20001])
def test_padding_of_norms_without_a_finite_root(cols):
    """eps = 0: a row of zeros has 0 * inf, one whose squares underflow t * inf; rows with NaN and infinity."""
    d = device()
    x = np.ones((5, cols), np.float32)
    x[0] = 0
    x[1] = 1e-25
    x[2, cols - 1] = np.nan
    x[3, 2] = np.inf
    t, (q, s) = up(x), d.e4m3(5, cols)
    filled(q)
    d.rmsnorm_rows(5, cols, t, up(np.ones(cols)), 0.0, q=q, q_scale=s)
    got, sc = get_bytes(q, 5, MB.e4m3_ld(cols)), s.read().reshape(5, -1)
    assert not got[:, cols:].any()
    assert np.all((got[:3, :cols] & 0x7F) == 0x7F) and np.isnan(sc[[0, 2]]).all() and np.isposinf(sc[1]).all()
    # the root of a row with an infinity is 0: the infinity gives NaN, which takes its group, the others give 0
    assert np.all((got[3, :128] & 0x7F) == 0x7F) and not (got[3, 128:] & 0x7F).any()
    assert np.all(got[4, :cols] == 0x7E) and np.isfinite(sc[4]).all()


@pytest.mark.parametrize("block", [True, False])
@pytest.mark.parametrize("m,k,n", [(2, 512, 64), (20, 512, 96), (60, 300, 200), (140, 512, 300), (700, 640, 5000)])
def test_products_of_whole_numbers_are_exact(m, k, n, block):
    """0, +-1, 2, 3 and scales of powers of two: every product and sum is a whole number below 2^24 times a
    power of two, so f32 holds it whatever the order, and the result is equal bit for bit."""
    d = device()
    g = np.random.default_rng([0xE7, m])
    codes = np.array([0x00, 0x38, 0x40, 0x44, 0xB8, 0xC0], np.uint8)
    ld = MB.e4m3_ld(k)

    def operand(rows, blocks):
        q = np.zeros((rows, ld), np.uint8)
        q[:, :k] = codes[g.integers(0, len(codes), (rows, k))]
        s = 2.0 ** g.integers(0, 3, (-(-rows // 128) if blocks else rows, ld // 128))
        full = np.repeat(s, 128, 0)[:rows] if blocks else s
        return q, s.astype(np.float32), VALUES[q].astype(np.float64) * np.repeat(full, 128, 1)

    xq, xs, x = operand(m, False)
    yq, ys, y = operand(n, block)
    r = d.tensor((n, m))
    d.matmul_e4m3(m, k, n, r, up(xq.view(np.float32)), up(xs), up(yq.view(np.float32)), up(ys), y_block=block)
    want = x @ y.T  # at most 640 * 9 * 16, exact
    assert np.array_equal(r.read().reshape(m, n), want.astype(np.float32))
