"""Head norm and rotation, the paged cache and attention over it, on the GPU against 64 bits.

U = 2^-24 is half an f32 step relative to the value; tolerances count roundings (attention's are derived in
attention_ref.py)."""
import math

import numpy as np
import pytest

import attention_ref as R
import mag_b200 as MB
from attention_ref import U, VALUES
from gpu_util import device
from test_gpu_lm_graphs import capture

pytestmark = pytest.mark.gpu

EPS = 1e-6


def rng(*key):
    return np.random.default_rng([0xA7, *key])


def up(a):
    a = np.ascontiguousarray(a, np.float32)
    t = device().tensor((max(1, a.size),))
    if a.size:
        t.write(a.reshape(-1))
    return t


def ints(a):
    return device().ids(np.asarray(a))


def blank(*shape):
    """A result buffer full of NaN, so that values left unwritten show."""
    return up(np.full(shape, np.nan, np.float32))


def get(t, *shape):
    return t.read()[:int(np.prod(shape))].reshape(shape)


def raw(t):
    return t.read().view(np.uint8)


def strided(a, stride, at=0):
    """Rows of a [rows][width] at a stride, `at` values into the buffer; NaN between them."""
    b = np.full(at + a.shape[0] * stride, np.nan, np.float32)
    b[at:].reshape(a.shape[0], stride)[:, :a.shape[1]] = a
    return b


def rows_of(flat, rows, stride, width, at=0):
    return flat[at:at + rows * stride].reshape(rows, stride)[:, :width]


# ------------------------------------------------------------------ norm and rotation of heads
HEADS = [  # rows, heads, dim, rot, pairs, norm, extra stride, offset
    (1, 1, 8, 8, False, True, 0, 0), (3, 2, 16, 16, True, True, 0, 0), (5, 12, 80, 16, True, True, 0, 0), (7, 5, 64, 64, False, True, 4, 0),
    (2, 3, 64, 32, False, False, 0, 0), (9, 32, 128, 128, False, True, 0, 0), (4, 7, 128, 64, True, True, 3, 1), (6, 3, 96, 96, False, True, 0, 3),
    (3, 4, 256, 256, False, True, 0, 0), (3, 4, 256, 128, False, True, 8, 0), (2, 5, 200, 200, True, False, 0, 0), (2, 3, 192, 96, False, True, 1, 0),
    (300, 3, 48, 24, False, True, 0, 0), (150, 9, 128, 128, False, False, 0, 0), (4, 2, 72, 0, False, True, 0, 0), (33, 33, 32, 8, True, True, 0, 0)]


def head_inputs(rows, heads, dim, rot, norm, key=0):
    g = rng(rows, heads, dim, key)
    x = (g.normal(0, 1, (rows, heads, dim)) * np.exp(g.normal(0, 0.7, dim))).astype(np.float32)
    pos = g.integers(0, 200000, rows)
    pos[0] = (1 << 31) - 1
    w = (1 + 0.3 * g.normal(0, 1, dim)).astype(np.float32) if norm else None
    return g, x, pos, MB.rope_frequencies(rot, 500000.0), w


def rotation(pos, freq, rot, pairs, mag=1.0):
    return MB.Rotation(ints(pos), up(freq), rot, interleaved=pairs, magnitude=mag) if rot else None


@pytest.mark.parametrize("rows,heads,dim,rot,pairs,norm,extra,at", HEADS)
def test_rotate_heads(rows, heads, dim, rot, pairs, norm, extra, at):
    d = device()
    _, x, pos, freq, w = head_inputs(rows, heads, dim, rot, norm)
    n, mag = heads * dim, 1.0 if rows % 2 else 1.25
    s = n + extra
    xb, yb = up(strided(x.reshape(rows, n), s, at)), blank(at + rows * s)
    rs = blank(rows, heads) if norm else None
    d.rotate_heads(rows, heads, dim, yb.data_ptr + 4 * at, xb.data_ptr + 4 * at, w=up(w) if norm else None, eps=EPS, rstd=rs,
                   rotation=rotation(pos, freq, rot, pairs, mag), x_stride=s, y_stride=s)
    v, rstd = R.norm(x, w, EPS) if norm else (x, None)
    want, size = R.turn(v, pos, freq, rot, pairs, mag)
    y = yb.read()
    got = rows_of(y, rows, s, n, at).reshape(rows, heads, dim)
    # the sum of squares: at most 8 terms a lane and 5 joins, half of it in the root; root, products, angle, turn
    assert np.all(np.abs(got - want) <= (7 + 10) * U * size)
    if norm:
        assert np.all(np.abs(get(rs, rows, heads) - rstd) <= 9 * U * rstd)
    if extra:
        assert np.isnan(y[at:].reshape(rows, s)[:, n:]).all()
    # in place
    d.rotate_heads(rows, heads, dim, xb.data_ptr + 4 * at, xb.data_ptr + 4 * at, w=up(w) if norm else None, eps=EPS,
                   rotation=rotation(pos, freq, rot, pairs, mag), x_stride=s, y_stride=s)
    assert np.array_equal(rows_of(xb.read(), rows, s, n, at), rows_of(y, rows, s, n, at))


def test_rotations_of_far_positions():
    """Every frequency of the table at the ends of int32 and around: the turn's fraction survives."""
    d = device()
    pos = np.array([-(1 << 31), -(1 << 31) + 1, -70001, -1, 0, 1, 2, 1 << 20, 16777217, (1 << 31) - 2, (1 << 31) - 1], np.int64)
    freq = np.concatenate([MB.rope_frequencies(64, 10000.0), np.float32([1.0, 3.1415927, 1.5707964, 0.7853982] * 8)])
    x = np.zeros((len(pos), 1, 128), np.float32)
    x[..., :64] = 1.0
    y = blank(len(pos), 128)
    d.rotate_heads(len(pos), 1, 128, y, up(x), rotation=rotation(pos, freq, 128, False))
    want, _ = R.turn(x, pos, freq, 128, False)
    assert np.all(np.abs(get(y, len(pos), 1, 128) - want) <= 6 * U)


def test_special_values_stay_in_their_heads():
    d = device()
    x = np.ones((2, 3, 64), np.float32)
    x[0, 1, 3], x[1, 2, 60] = np.nan, np.inf  # value 60 lies behind the rotated part
    y = blank(2, 192)
    d.rotate_heads(2, 3, 64, y, up(x), rotation=rotation([5, 9], MB.rope_frequencies(32), 32, False))
    bad = ~np.isfinite(get(y, 2, 3, 64))
    assert set(zip(*np.nonzero(bad))) == {(0, 1, 3), (0, 1, 19), (1, 2, 60)}
    x[:] = 0.0
    d.rotate_heads(2, 3, 64, y, up(x), w=up(np.ones(64)), eps=0.0)  # zeros without eps: 0 * infinity
    assert np.isnan(get(y, 2, 192)).all()
    d.rotate_heads(2, 3, 64, y, up(x), w=up(np.ones(64)), eps=EPS)
    assert not get(y, 2, 192).any()


@pytest.mark.parametrize("rows,heads,dim,rot,pairs,norm,extra,at", HEADS + [(1999, 5, 128, 128, False, True, 0, 0), (900, 2, 64, 64, True, True, 0, 0)])
def test_rotate_heads_backward(rows, heads, dim, rot, pairs, norm, extra, at):
    d = device()
    g, x, pos, freq, w = head_inputs(rows, heads, dim, rot, norm, 1)
    n, mag = heads * dim, 1.25
    s = n + extra
    dy = g.normal(0, 1, (rows, heads, dim)).astype(np.float32)
    rot_ = rotation(pos, freq, rot, pairs, mag)
    dyb, dxb = up(strided(dy.reshape(rows, n), s, at)), blank(at + rows * s)
    u, size = R.turn(dy, pos, freq, rot, pairs, mag, back=True)
    if not norm:
        d.rotate_heads_backward(rows, heads, dim, dxb.data_ptr + 4 * at, None, dyb.data_ptr + 4 * at, rotation=rot_, dx_stride=s, dy_stride=s)
        assert np.all(np.abs(rows_of(dxb.read(), rows, s, n, at).reshape(x.shape) - u) <= 6 * U * size)
        return
    rstd = R.norm(x, w, EPS)[1].astype(np.float32)
    xb, dw = up(strided(x.reshape(rows, n), s, at)), blank(dim)
    args = dict(x=xb.data_ptr + 4 * at, w=up(w), rstd=up(rstd), rotation=rot_, dx_stride=s, dy_stride=s, x_stride=s)
    d.rotate_heads_backward(rows, heads, dim, dxb.data_ptr + 4 * at, dw, dyb.data_ptr + 4 * at, **args)
    r, X, W = rstd.astype(np.float64)[..., None], x.astype(np.float64), w.astype(np.float64)
    c = (u * W * X).mean(-1, keepdims=True) * r * r
    want = r * (u * W - X * c)
    mean = (size * np.abs(W * X)).mean(-1, keepdims=True) * r * r
    got = dxb.read()
    # u: 6 roundings; the mean: 8 terms a lane, 5 joins and a few factors
    assert np.all(np.abs(rows_of(got, rows, s, n, at).reshape(x.shape) - want) <= U * r * (9 * size * np.abs(W) + 26 * np.abs(X) * mean))
    terms = u * X * r
    # a lane adds one term for each head row of its group (at most rows * heads / (8 * blocks) + heads of them); blocks are
    # joined in at most 16 + 14 + 32 further additions
    each = min(rows * heads, rows * heads / (8 * min(444, -(-rows // 4))) + 4 * heads)
    assert np.all(np.abs(get(dw, dim) - terms.sum((0, 1))) <= (each + 70) * U * (size * np.abs(X) * r).sum((0, 1)))
    first = get(dw, dim).copy()
    d.rotate_heads_backward(rows, heads, dim, dyb.data_ptr + 4 * at, dw, dyb.data_ptr + 4 * at, **args)  # over dy, and the same again
    assert np.array_equal(rows_of(dyb.read(), rows, s, n, at), rows_of(got, rows, s, n, at)) and np.array_equal(get(dw, dim), first)


def test_gradient_against_differences():
    """The 64-bit formula that the kernels are held to, against differences of the 64-bit forward pass."""
    g, x, pos, freq, w = head_inputs(2, 2, 16, 8, True, 2)
    x, w, dy = x.astype(np.float64), w.astype(np.float64), g.normal(0, 1, x.shape)

    def f(x, w):
        return (R.turn(R.norm(x, w, EPS)[0], pos, freq, 8, False, 1.25)[0] * dy).sum()

    d = device()
    dx, dw = blank(2, 32), blank(16)
    rstd = R.norm(x, w, EPS)[1]
    d.rotate_heads_backward(2, 2, 16, dx, dw, up(dy), x=up(x), w=up(w), rstd=up(rstd), rotation=rotation(pos, freq, 8, False, 1.25))
    h = 1e-5
    for got, a, shape in ((get(dx, 2, 2, 16), x, x.shape), (get(dw, 16), w, w.shape)):
        for at in np.ndindex(*shape):
            hi, lo = a.copy(), a.copy()
            hi[at] += h
            lo[at] -= h
            diff = (f(hi, w) - f(lo, w) if a is x else f(x, hi) - f(x, lo)) / (2 * h)
            assert abs(got[at] - diff) <= 1e-4 * max(1.0, abs(diff)), at


def test_backward_of_no_rows():
    d = device()
    dw = blank(64)
    d.rotate_heads_backward(0, 2, 64, up(0), dw, up(0), x=up(0), w=up(np.ones(64)), rstd=up(0))
    assert not get(dw, 64).any()


# ------------------------------------------------------------------ the cache
def random_cache(pages, heads, dim, page, key=0, spread=0.4):
    """A cache whose every slot is written, and its values [pages * page][heads][dim] in 64 bits."""
    g = rng(pages, heads, dim, page, key)
    c = device().kv_cache(pages, heads, dim, page)
    out = []
    for t, ts in ((c.k, c.k_scale), (c.v, c.v_scale)):
        b = g.integers(0, 256, (pages, heads, page, dim)).astype(np.uint8)
        b[(b & 0x7F) == 0x7F] = 0
        s = (np.exp(g.normal(0, spread, (pages, heads, page))) / 150.0).astype(np.float32)
        t.write(b.reshape(-1).view(np.float32))
        ts.write(s)
        v = VALUES[b] * s.astype(np.float64)[..., None]
        out.append(v.transpose(0, 2, 1, 3).reshape(pages * page, heads, dim))
    return c, out[0], out[1]


def cache_bytes(c):
    shape = (c.pages, c.heads, c.page_size)
    return [raw(c.k).reshape(*shape, c.head_dim), get(c.k_scale, *shape), raw(c.v).reshape(*shape, c.head_dim), get(c.v_scale, *shape)]


def half_step(v):
    _, e = np.frexp(np.minimum(np.abs(v), 448.0))
    return 2.0 ** (np.maximum(e - 4, -9) - 1)


def check_rows(q, s, v, err):
    """e4m3 rows q with scales s against the values v, known within err."""
    top, slack = np.abs(v).max(-1), err.max(-1)
    want = np.maximum(top, 2.0 ** -100) / 448.0
    assert np.all(np.abs(s - want) <= want * 2 * U + slack / 448.0)
    t = v / s.astype(np.float64)[..., None]
    e = err / s.astype(np.float64)[..., None] + np.abs(t) * 2 * U
    assert np.all(np.abs(VALUES[q] - t) <= half_step(np.abs(t) + e) + e)


WRITES = [  # rows, q_heads, heads, dim, page, rot, pairs, norm, extra
    (1, 4, 2, 64, 16, 64, False, True, 0), (8, 32, 8, 128, 16, 128, False, True, 0), (37, 6, 3, 96, 32, 48, False, True, 0),
    (5, 0, 2, 16, 16, 16, True, True, 0), (70, 5, 5, 80, 64, 16, True, False, 4), (200, 8, 8, 128, 128, 128, False, False, 1),
    (33, 7, 1, 112, 1024, 56, False, True, 0), (300, 3, 1, 48, 256, 0, False, True, 0), (150, 40, 8, 64, 64, 64, False, True, 0)]


@pytest.mark.parametrize("rows,qh,heads,dim,page,rot,pairs,norm,extra", WRITES)
def test_kv_write(rows, qh, heads, dim, page, rot, pairs, norm, extra):
    d = device()
    g, x, pos, freq, k_w = head_inputs(rows, qh + 2 * heads, dim, rot, norm, 3)
    q_w = (1 + 0.3 * g.normal(0, 1, dim)).astype(np.float32) if norm and qh else None
    pages = -(-rows // page) + 2
    c, _, _ = random_cache(pages, heads, dim, page, 1)
    before = [a.copy() for a in cache_bytes(c)]
    slot = g.permutation(pages * page)[:rows].astype(np.int64)
    skip = g.random(rows) < (0.2 if rows > 1 else 0.0)
    slot[skip] = g.choice([-1, -(1 << 31), pages * page, (1 << 31) - 1], skip.sum())
    width = (qh + 2 * heads) * dim
    s = width + extra
    fused = up(strided(x.reshape(rows, width), s))
    q_out = blank(rows, max(1, qh) * dim)
    at = fused.data_ptr
    d.kv_write(c, rows, ints(slot), at + 4 * qh * dim, at + 4 * (qh + heads) * dim, k_w=up(k_w) if norm else None, q=at if qh else None,
               q_out=q_out if qh else None, q_heads=qh, q_w=up(q_w) if norm and qh else None, eps=EPS,
               rotation=rotation(pos, freq, rot, pairs), k_stride=s, v_stride=s, q_stride=s)
    q, k, v = x[:, :qh], x[:, qh:qh + heads], x[:, qh + heads:].astype(np.float64)
    if norm:
        q, k = R.norm(q, q_w, EPS)[0] if qh else q, R.norm(k, k_w, EPS)[0]
    if qh:
        want, size = R.turn(q, pos, freq, rot, pairs)
        assert np.all(np.abs(get(q_out, rows, qh, dim) - want) <= 17 * U * size)
    k, size = R.turn(k, pos, freq, rot, pairs)
    after = cache_bytes(c)
    touched = np.zeros((pages, page), bool)
    put = slot[~skip]
    touched[put // page, put % page] = True
    for a, b in zip(after, before):
        assert np.array_equal(a.transpose(0, 2, 1, *range(3, a.ndim))[~touched], b.transpose(0, 2, 1, *range(3, b.ndim))[~touched])
    check_rows(after[0][put // page, :, put % page], after[1][put // page, :, put % page], k[~skip], 17 * U * size[~skip])
    check_rows(after[2][put // page, :, put % page], after[3][put // page, :, put % page], v[~skip], np.zeros_like(v[~skip]))


def test_special_rows_in_the_cache():
    d = device()
    c = d.kv_cache(1, 2, 32, 16)
    k, v = np.ones((4, 2, 32), np.float32), np.zeros((4, 2, 32), np.float32)
    k[0, 0, 5], k[1, 1, 31], v[2, 0, 0], v[3, 1, 1] = np.nan, -np.inf, 3e38, 2.0 ** -120
    d.kv_write(c, 4, ints([0, 1, 2, 3]), up(k), up(v))
    kb, ks, vb, vs = cache_bytes(c)
    assert np.isnan(ks[0, 0, 0]) and np.isnan(ks[0, 1, 1]) and not kb[0, 0, 0].any() and not kb[0, 1, 1].any()
    assert np.all(kb[0, 1, 0] == 0x7E) and ks[0, 1, 0] == np.float32(1) * np.float32(1 / 448)
    assert vb[0, 0, 2, 0] == 0x7E and not vb[0, 1, 3].any() and vs[0, 1, 3] == np.float32(2.0 ** -100) * np.float32(1 / 448)
    assert not kb[0, :, 4:].any() and not ks[0, :, 4:].any()  # never written: zeros
    ko, vo = blank(5, 64), blank(5, 64)
    d.kv_read(c, 5, ints([0, 3, 16, -1, 9]), k=ko, v=vo)
    ko, vo = get(ko, 5, 2, 32), get(vo, 5, 2, 32)
    assert np.isnan(ko[0, 0]).all() and np.all(ko[0, 1] == ko[0, 1, 0]) and not ko[2:].any() and not vo[2:].any()


@pytest.mark.parametrize("rows,heads,dim,page,extra", [(1, 1, 16, 16, 0), (300, 2, 96, 16, 0), (77, 8, 128, 64, 5), (1000, 3, 64, 32, 0), (5, 5, 112, 1024, 4)])
def test_kv_read(rows, heads, dim, page, extra):
    d = device()
    pages = max(2, -(-rows // page) // 2)
    c, k, v = random_cache(pages, heads, dim, page)
    slot = rng(rows).integers(0, pages * page, rows)  # some slots twice
    n = heads * dim
    ko, vo = blank(rows, n + extra), blank(rows, n)
    d.kv_read(c, rows, ints(slot), k=ko, v=vo, k_stride=n + extra)
    # one product of an f32 and an e4m3 value, rounded
    assert np.array_equal(get(ko, rows, n + extra)[:, :n].reshape(rows, heads, dim), k[slot].astype(np.float32))
    assert np.array_equal(get(vo, rows, heads, dim), v[slot].astype(np.float32))
    assert np.isnan(get(ko, rows, n + extra)[:, n:]).all()
    only = blank(rows, n)
    d.kv_read(c, rows, ints(slot), v=only)
    assert np.array_equal(only.read(), vo.read())
    d.kv_read(c, rows, ints(slot), k=only)
    assert np.array_equal(get(only, rows, heads, dim), k[slot].astype(np.float32))


# ------------------------------------------------------------------ attention
class Batch:
    """Sequences [(new, length), ..] over a cache with shuffled pages."""

    def __init__(self, seqs, q_heads, heads, dim, page, *, window=0, key=0, pad=0, extra=0, scale=None, q_scale=1.0, before=0):
        g = rng(len(seqs), q_heads, dim, page, key)
        self.seqs, self.heads, self.dim, self.page, self.window = seqs, (q_heads, heads), dim, page, window
        need = [-(-l // page) for _, l in seqs]
        self.pages = sum(need) + 2
        order = g.permutation(self.pages)
        self.table = np.full((len(seqs), max(1, *need) + 1), -1, np.int64)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        self.cache, self.k, self.v = random_cache(self.pages, heads, dim, page, key)
        self.start = before + np.cumsum([0] + [n for n, _ in seqs])
        self.rows = int(self.start[-1]) + pad
        self.q = (g.normal(0, 1, (self.rows, q_heads, dim)) * np.exp(g.normal(0, 0.5, (self.rows, q_heads, 1))) * q_scale).astype(np.float32)
        self.scale = float(np.float32(1.3 / math.sqrt(dim) if scale is None else scale))
        self.max_new = max([n for n, _ in seqs] + [0])
        self.stride = q_heads * dim + extra

    def device_args(self):
        self.tq = up(strided(self.q.reshape(self.rows, -1), self.stride))
        self.tt, self.ts, self.tl = ints(self.table), ints(self.start), ints([l for _, l in self.seqs])
        self.out, self.lse = blank(self.rows, self.stride), blank(self.rows, self.heads[0])

    def call(self, max_new=None):
        device().attention_paged(self.cache, self.rows, self.heads[0], self.out, self.tq, self.tt, self.ts, self.tl, len(self.seqs),
                                 self.table.shape[1], max_new=self.max_new if max_new is None else max_new, scale=self.scale,
                                 window=self.window, lse=self.lse, q_stride=self.stride, out_stride=self.stride)

    def run(self, max_new=None):
        self.device_args()
        self.call(max_new)
        return self.results()

    def results(self):
        o = get(self.out, self.rows, self.stride)
        width = self.heads[0] * self.dim
        assert np.isnan(o[:, width:]).all()
        return o[:, :width].reshape(self.rows, self.heads[0], self.dim), get(self.lse, self.rows, self.heads[0])

    def want(self, i):
        n, length = self.seqs[i]
        j = np.arange(length)
        page = self.table[i][j // self.page]
        ok = (page >= 0) & (page < self.pages)
        at = np.where(ok, page, 0) * self.page + j % self.page
        return R.attention(self.q[self.start[i]:self.start[i + 1]].astype(np.float64), self.k[at], self.v[at], self.scale, n, length,
                           self.window, ok)

    def check(self, got=None):
        o, l = self.run() if got is None else got
        seen = np.zeros(self.rows, bool)
        for i in range(len(self.seqs)):
            rows = slice(self.start[i], self.start[i + 1])
            seen[rows] = True
            out, lse, tol, ltol = self.want(i)
            assert np.all(np.abs(o[rows] - out) <= tol), (i, self.seqs[i], np.nanmax(np.abs(o[rows] - out) / np.maximum(tol, 1e-30)))
            none = np.isneginf(lse)
            assert np.all(np.isneginf(l[rows][none])) and not o[rows][none].any()
            assert np.all(np.abs(l[rows][~none] - lse[~none]) <= ltol[~none]), (i, self.seqs[i])
        assert np.isnan(o[~seen]).all() and np.isnan(l[~seen]).all()


@pytest.mark.parametrize("group", [1, 2, 4, 5, 8, 9, 16, 17])
@pytest.mark.parametrize("dim", [16, 64, 80, 128])
def test_single_tokens(group, dim):
    Batch([(1, 1), (1, 15), (1, 16), (1, 17), (1, 129), (1, 700)], 2 * group, 2, dim, 16).check()


@pytest.mark.parametrize("page", [16, 64, 256, 1024])
def test_single_tokens_pages(page):
    Batch([(1, n) for n in (1, page - 1, page, page + 1, 2 * page + 5, 1500)], 8, 2, 96, page).check()


@pytest.mark.parametrize("new,length", [(2, 2), (3, 40), (16, 16), (17, 300), (33, 1000), (64, 64), (128, 129), (130, 500), (200, 200)])
@pytest.mark.parametrize("q_heads,heads,dim,page", [(4, 1, 128, 16), (6, 2, 64, 64), (5, 1, 96, 32)])
def test_chunks(new, length, q_heads, heads, dim, page):
    Batch([(new, length)], q_heads, heads, dim, page).check()


@pytest.mark.parametrize("dim", [16, 48, 64, 112, 128])
def test_ragged_batch(dim):
    """Single tokens, chunks, prompts, a sequence without new tokens and one without any, in one call."""
    Batch([(1, 300), (40, 40), (0, 50), (1, 1), (150, 333), (0, 0), (3, 3), (70, 2000)], 10, 2, dim, 32).check()


@pytest.mark.parametrize("q_heads,heads", [(1, 1), (12, 12), (64, 1), (40, 8), (130, 1), (3, 1)])
def test_head_layouts(q_heads, heads):
    Batch([(1, 200), (30, 77), (1, 64)], q_heads, heads, 64, 16).check()


@pytest.mark.parametrize("window", [1, 2, 16, 100, 128, 1000, 5000])
@pytest.mark.parametrize("new", [1, 60])
def test_windows(new, window):
    Batch([(new, 900), (new, 60), (min(new, 9), 130)], 8, 2, 64, 16, window=window).check()


def test_long_sequences():
    """Lengths that many blocks share, single tokens and a chunk, next to short ones."""
    Batch([(1, 20011), (1, 5), (1, 3000)], 8, 1, 128, 64).check()
    Batch([(20, 9001), (1, 5)], 8, 1, 64, 128).check()


def test_many_sequences():
    Batch([(1, 1 + (37 * i) % 90) for i in range(1100)], 2, 2, 16, 16).check()


def test_many_sequences_of_chunks():
    Batch([(1 + i % 19, 20 + (37 * i) % 90) for i in range(600)], 2, 1, 16, 16).check()


@pytest.mark.parametrize("count,longest,q_heads,heads", [(1, 500, 4, 2), (3, 300, 8, 8), (7, 700, 2, 1), (40, 300, 16, 4), (150, 260, 3, 3), (400, 130, 4, 1),
                                                         (2, 9000, 40, 4), (5, 2100, 36, 4)])
def test_shares_that_end_anywhere(count, longest, q_heads, heads):
    """Sequences of all lengths, so that the blocks' shares end at items' beginnings, near them and within."""
    g = rng(count, longest)
    Batch([(1, int(n)) for n in g.integers(1, longest, count)], q_heads, heads, 64, 16).check()


def test_strides_and_rows_outside():
    """Padded rows, rows before the first and behind the last sequence: left as they were."""
    for seqs in ([(1, 40), (1, 9)], [(30, 50), (1, 20)]):
        Batch(seqs, 6, 2, 64, 16, extra=7, pad=5, before=3).check()
        Batch(seqs, 6, 2, 64, 16, extra=4, pad=0, before=0).check()


def test_padded_batch():
    """Every sequence has room for max_new rows, but most have fewer; rows = seqs * max_new all the same."""
    b = Batch([(1, 30), (40, 40), (2, 80)], 4, 2, 64, 16, pad=3 * 40 - 43)
    assert b.rows == len(b.seqs) * b.max_new
    b.check()


@pytest.mark.parametrize("new", [1, 40])
def test_rows_that_see_nothing(new):
    """New tokens that are not in the cache (length below the new tokens) and lengths of zero and below."""
    b = Batch([(new, max(1, new // 2)), (new, 0), (new, 33 + new)], 4, 2, 64, 16)
    b.check()
    n = b.seqs
    b.device_args()
    b.tl = ints([n[0][1], -7, n[2][1]])
    b.call()
    b.check(b.results())


@pytest.mark.parametrize("new", [1, 25])
def test_pages_that_do_not_exist(new):
    """Entries outside the cache hide their tokens; a sequence of such pages alone sees nothing."""
    b = Batch([(new, 400), (new, 40), (new, 100)], 4, 2, 64, 16)
    b.table[0, [0, 3, 7, 24]] = [-1, b.pages, (1 << 31) - 1, -(1 << 31)]
    b.table[1, :] = -1
    b.check()


@pytest.mark.parametrize("new", [1, 25])
def test_a_length_past_the_table(new):
    b = Batch([(new, 16 * 7)], 4, 2, 64, 16)
    b.table = b.table[:, :7]
    b.device_args()
    b.tl = ints([1 << 30])
    b.call()
    b.check(b.results())


@pytest.mark.parametrize("new", [1, 25])
def test_starts_out_of_order_stay_in_bounds(new):
    """Starts that fall or lie outside the rows: no row outside is touched, the good sequence is right."""
    b = Batch([(new, 50), (new, 60), (new, 70)], 4, 2, 64, 16)
    b.device_args()
    b.ts = ints([-5, -9, new, 1 << 30])
    b.call()
    o, l = b.results()
    # sequence 1 has the rows 0 .. new - 1, sequence 2 all the rest (of which max_new are taken)
    out, lse, tol, ltol = R.attention(b.q[:new].astype(np.float64), b.k[(b.table[1][np.arange(60) // 16] * 16 + np.arange(60) % 16)],
                                      b.v[(b.table[1][np.arange(60) // 16] * 16 + np.arange(60) % 16)], b.scale, new, 60, 0)
    assert np.all(np.abs(o[:new] - out) <= tol)
    assert np.isnan(o[2 * new:]).all()


@pytest.mark.parametrize("new", [1, 40])
def test_more_new_tokens_than_promised(new):
    """Rows past max_new are left; those before are as ever."""
    b = Batch([(new + 5, 200), (new, 90)], 4, 2, 64, 16)
    o, l = b.run(max_new=new)
    out, lse, tol, ltol = b.want(0)
    assert np.all(np.abs(o[:new] - out[:new]) <= tol[:new]) and np.isnan(o[new:new + 5]).all() and np.isnan(l[new:new + 5]).all()
    out, lse, tol, ltol = b.want(1)
    assert np.all(np.abs(o[new + 5:] - out) <= tol)


@pytest.mark.parametrize("new", [1, 33])
def test_unwritten_slots_and_nan_keys(new):
    """NaN bytes and scales behind the last token, in pages that no sequence has and before the window do not show; a NaN
    key or value shows in the rows that see it and in no other; a NaN query in its own row."""
    b = Batch([(new, 70), (new, 100)], 4, 2, 64, 16, window=50)
    kb, ks, vb, vs = [a.copy() for a in cache_bytes(b.cache)]
    used = np.zeros((b.pages, 16), bool)
    for i, (n, length) in enumerate(b.seqs):
        j = np.arange(max(0, length - n + 1 - 50), length)
        used[b.table[i][j // 16], j % 16] = True
    for a, s in ((kb, ks), (vb, vs)):
        a.transpose(0, 2, 1, 3)[~used] = 0x7F
        s.transpose(0, 2, 1)[~used] = np.nan
    hole = b.table[1][99 // 16], 1, 99 % 16  # the last token's value of kv head 1, NaN as kv_write leaves it
    vb[hole], vs[hole] = 0, np.nan
    for t, a in zip((b.cache.k, b.cache.k_scale, b.cache.v, b.cache.v_scale), (kb, ks, vb, vs)):
        t.write(a.reshape(-1).view(np.float32))
    b.q[0, 3, 7] = np.nan
    o, l = b.run()
    nan = np.zeros(o.shape[:2], bool)
    nan[0, 3] = True
    nan[2 * new - 1, 2:] = True  # the query heads of kv head 1, in the one row that sees token 99
    assert np.array_equal(np.isnan(o).any(-1), nan) and np.array_equal(np.isnan(o).all(-1), nan)
    for i in range(2):
        rows = slice(b.start[i], b.start[i + 1])
        b.q[0, 3, 7] = 0.0
        out, lse, tol, ltol = b.want(i)
        good = ~nan[rows]
        assert np.all(np.abs(o[rows] - out)[good] <= tol[good])


@pytest.mark.parametrize("new", [1, 33])
def test_large_and_small_values(new):
    """Queries of 2^40 and 2^-60, keys' scales to match, values' scales over 80 powers of two, logits in the hundreds."""
    b = Batch([(new, 150), (new, 40)], 4, 2, 64, 16)
    g = rng(new, 77)
    b.q *= np.float32(2.0) ** g.integers(-60, 41, (b.rows, 4, 1)).astype(np.float32)
    b.check()
    b = Batch([(new, 150), (new, 40)], 4, 2, 64, 16, scale=60.0)
    b.check()
    b = Batch([(new, 150), (new, 40)], 4, 2, 64, 16, scale=0.0)
    b.check()
    b = Batch([(new, 300)], 4, 2, 64, 16)
    s = get(b.cache.v_scale, b.pages, 2, 16) * np.float32(2.0) ** g.integers(-60, 21, (b.pages, 2, 16)).astype(np.float32)
    b.v = b.v * (s.astype(np.float64) / get(b.cache.v_scale, b.pages, 2, 16)).transpose(0, 2, 1).reshape(-1, 2, 1)
    b.cache.v_scale.write(s)
    b.check()


def test_values_far_behind_the_largest_weight():
    """One token takes nearly all the weight and has no value; what the others bring is kept to f32 precision."""
    b = Batch([(1, 600)], 1, 1, 64, 16)
    kb, ks, vb, vs = [a.copy() for a in cache_bytes(b.cache)]
    p, r = b.table[0][2], 5
    vb[p, 0, r] = 0
    b.cache.v.write(vb.reshape(-1).view(np.float32))
    b.v[p * 16 + r] = 0.0
    b.q[:] = 0.0
    b.q[0, 0, 3] = 1.0
    kb[..., 3] = 0
    kb[p, 0, r, 3] = 0x7E
    b.cache.k.write(kb.reshape(-1).view(np.float32))
    b.k[..., 3] = 0.0
    b.k[p * 16 + r, 0, 3] = 448.0 * float(ks[p, 0, r])
    b.scale = 14.0 / b.k[p * 16 + r, 0, 3]  # the others weigh 2^-20 of the one
    b.scale = float(np.float32(b.scale))
    b.check()


def test_repeated_calls_are_the_same_bits():
    b = Batch([(1, 3000), (40, 700), (1, 17)], 8, 2, 128, 32)
    first = b.run()
    for _ in range(3):
        again = b.run()
        assert all(np.array_equal(x.view(np.uint32), y.view(np.uint32)) for x, y in zip(first, again))


def test_pages_shared_by_sequences():
    """A common prefix lies in the cache once."""
    b = Batch([(1, 100), (30, 130), (1, 64)], 4, 2, 64, 16)
    b.table[1, :4] = b.table[2, :4] = b.table[0, :4]
    b.check()


def test_offsets_past_32_bits():
    """A cache of 4.6 GB of keys and as much of values: pages behind 2^32 bytes, read and written."""
    d = device()
    page, heads, dim = 1024, 8, 128
    pages = (1 << 32) // (page * heads * dim) + 300
    c = d.kv_cache(pages, heads, dim, page)
    g = rng(99)
    rows = 40
    k, v = (g.normal(0, 1, (rows, heads, dim)).astype(np.float32) for _ in range(2))
    last = pages - 1
    slot = last * page + np.arange(rows) + 7
    d.kv_write(c, rows, ints(slot), up(k), up(v))
    ko, vo = blank(rows, heads * dim), blank(rows, heads * dim)
    d.kv_read(c, rows, ints(slot), k=ko, v=vo)
    ko, vo = get(ko, rows, heads, dim).astype(np.float64), get(vo, rows, heads, dim).astype(np.float64)
    assert np.all(np.abs(ko - k) <= np.abs(k).max(-1, keepdims=True) * 2.0 ** -4)
    for new in (1, 20):
        q = g.normal(0, 1, (new, 16, dim)).astype(np.float32)
        out, lse = blank(new, 16 * dim), blank(new, 16)
        length = 7 + rows
        d.attention_paged(c, new, 16, out, up(q), ints([last]), ints([0, new]), ints([length]), 1, 1, max_new=new, scale=0.1, lse=lse)
        kk, vv = np.zeros((length, heads, dim)), np.zeros((length, heads, dim))
        kk[7:], vv[7:] = ko, vo
        want, wl, tol, ltol = R.attention(q.astype(np.float64), kk, vv, float(np.float32(0.1)), new, length, 0)
        assert np.all(np.abs(get(out, new, 16, dim) - want) <= tol) and np.all(np.abs(get(lse, new, 16) - wl) <= ltol)


# ------------------------------------------------------------------ graphs, and a run of them together
@pytest.mark.parametrize("seqs", [[(1, 900), (1, 40)], [(50, 300), (50, 77)], [(1, 500), (60, 60)]])
def test_replays_follow_the_lengths_on_the_device(seqs):
    """Two captured calls that live together, replayed in turn with other lengths between: the pages' table, the starts
    and the lengths are read by each replay, and the graphs share no scratch."""
    a, b = Batch(seqs, 8, 2, 64, 16, key=1), Batch(seqs, 8, 2, 64, 16, key=2)
    replays = []
    for x in (a, b):
        x.run()
        replays.append(capture(device(), [x.call]))
    for step in range(3):
        for x in (a, b):
            x.seqs = [(n, max(n, l - 13 * step)) for n, l in x.seqs]
            x.tl.write(np.array([l for _, l in x.seqs], np.int32).view(np.float32))
            for t in (x.out, x.lse):
                t.write(np.full(t.numel, np.nan, np.float32))
        replays[0](), replays[1](), replays[0]()
        for x in (a, b):
            x.check(x.results())


def test_captured_write_and_gradient():
    d = device()
    rows, qh, heads, dim = 6, 4, 2, 64
    g, x, pos, freq, w = head_inputs(rows, qh + 2 * heads, dim, dim, True, 5)
    pos[0] = 3
    c, fused, q_out, slot = d.kv_cache(2, heads, dim, 16), up(x), blank(rows, qh * dim), ints(np.arange(rows))
    rot, tw, width = rotation(pos, freq, dim, False), up(w), (qh + 2 * heads) * dim
    dy, dx, dw, rs = up(g.normal(0, 1, (rows, qh, dim))), blank(rows, qh * dim), blank(dim), blank(rows, qh)
    xq, y = up(x[:, :qh]), blank(rows, qh * dim)

    def calls():
        d.kv_write(c, rows, slot, fused.data_ptr + 4 * qh * dim, fused.data_ptr + 4 * (qh + heads) * dim, k_w=tw, q=fused.data_ptr,
                   q_out=q_out, q_heads=qh, q_w=tw, eps=EPS, rotation=rot, k_stride=width, v_stride=width, q_stride=width)
        d.rotate_heads(rows, qh, dim, y, xq, w=tw, eps=EPS, rstd=rs, rotation=rot)
        d.rotate_heads_backward(rows, qh, dim, dx, dw, dy, x=xq, w=tw, rstd=rs, rotation=rot)

    calls()
    d.sync()
    want = [t.read().copy() for t in (q_out, y, dx, dw, c.k, c.v, c.k_scale, c.v_scale)]
    assert np.array_equal(want[0], want[1])  # queries of the one pass and of the other
    replay = capture(d, [calls])
    for t in (q_out, y, dx, dw, c.k, c.v, c.k_scale, c.v_scale):
        t.fill_zero()
    replay()
    for t, a in zip((q_out, y, dx, dw, c.k, c.v, c.k_scale, c.v_scale), want):
        assert np.array_equal(t.read().view(np.uint32), a.view(np.uint32))


def test_a_prompt_and_its_tokens_one_by_one():
    """The path of a layer, in the order a model calls it: norm with e4m3 output, the product that makes queries, keys and
    values, their norms, rotation and cache, attention, the quantiser and the product that follows; once for a prompt of 37
    tokens in one call, and again token by token into other pages.  Each row's results agree to the products' rounding."""
    d = device()
    T, hidden, qh, heads, dim, page = 37, 256, 8, 2, 64, 16
    width = (qh + 2 * heads) * dim
    g = rng(123)
    x = up(g.normal(0, 1, (T, hidden)))
    nw, qw, kw = (up(1 + 0.2 * g.normal(0, 1, n)) for n in (hidden, dim, dim))
    wq, ws = d.e4m3(width, hidden, True)
    d.quantize_e4m3(hidden, width, up(g.normal(0, 1, (hidden, width)) / 16), wq, ws, block=True, transpose=True)
    oq, os_ = d.e4m3(hidden, qh * dim, True)
    d.quantize_e4m3(qh * dim, hidden, up(g.normal(0, 1, (qh * dim, hidden)) / 16), oq, os_, block=True, transpose=True)
    freq = up(MB.rope_frequencies(dim))
    cache = d.kv_cache(8, heads, dim, page)
    tables = [[5, 0, 3], [1, 7, 2]]

    def layer(first, n, table):
        hq, hs = d.e4m3(n, hidden)
        d.rmsnorm_rows(n, hidden, x.data_ptr + 4 * first * hidden, nw, EPS, q=hq, q_scale=hs)
        qkv, q, att, r = blank(n, width), blank(n, qh * dim), blank(n, qh * dim), blank(n, hidden)
        d.matmul_e4m3(n, hidden, width, qkv, hq, hs, wq, ws)
        at = np.arange(first, first + n)
        slot, pos = ints(np.array(table)[at // page] * page + at % page), ints(at)
        d.kv_write(cache, n, slot, qkv.data_ptr + 4 * qh * dim, qkv.data_ptr + 4 * (qh + heads) * dim, k_w=kw, q=qkv, q_out=q, q_heads=qh,
                   q_w=qw, eps=EPS, rotation=MB.Rotation(pos, freq, dim), k_stride=width, v_stride=width, q_stride=width)
        d.attention_paged(cache, n, qh, att, q, ints(table), ints([0, n]), ints([first + n]), 1, 3, max_new=n, scale=dim ** -0.5)
        aq, as_ = d.e4m3(n, qh * dim)
        d.quantize_e4m3(n, qh * dim, att, aq, as_)
        d.matmul_e4m3(n, qh * dim, hidden, r, aq, as_, oq, os_)
        return get(q, n, qh, dim), get(att, n, qh, dim), get(r, n, hidden)

    q, att, r = layer(0, T, tables[0])
    steps = [layer(t, 1, tables[1]) for t in range(T)]
    sizes = np.abs(att).max(-1, keepdims=True)
    for t in range(T):
        # the products' sums are formed in other orders for one row and for 37, so a key may round to its other e4m3 neighbour
        # (2^-3 of it apart): hold the results to one such step of one key in each head
        assert np.all(np.abs(steps[t][0][0] - q[t]) <= 2.0 ** -12 * np.abs(q[t]).max())
        assert np.all(np.abs(steps[t][1][0] - att[t]) <= 2.0 ** -3 * sizes[t] + 1e-6)
        assert np.all(np.abs(steps[t][2][0] - r[t]) <= 2.0 ** -3 * np.abs(r).max())
    # and attention of the prompt against 64 bits, from what the cache holds
    at = np.arange(T)
    slot = np.array(tables[0])[at // page] * page + at % page
    kb, ks, vb, vs = cache_bytes(cache)
    k, v = (VALUES[b[slot // page, :, slot % page]] * s[slot // page, :, slot % page].astype(np.float64)[..., None] for b, s in ((kb, ks), (vb, vs)))
    out, _, tol, _ = R.attention(q.astype(np.float64), k, v, dim ** -0.5, T, T, 0)
    assert np.all(np.abs(att - out) <= tol)
