"""Attention over the paged cache where values, their scales or the logits span far more than usual, against 64 bits.

U = 2^-24 is half an f32 step relative to the value; Batch and its tolerances are those of test_gpu_lm_attention.py, and
where a test needs a tighter one it is derived beside it."""
import numpy as np
import pytest

from attention_ref import U
from gpu_util import device
from test_gpu_lm_attention import Batch, blank, get, ints, up

pytestmark = pytest.mark.gpu

TOP = 0x7E  # the byte of 448


def set_values(b, value):
    """All of the cache's values to about `value`, b.v with them."""
    s = np.float32(value / 448.0)
    b.cache.v.write(np.full(b.cache.v.numel * 4, TOP, np.uint8).view(np.float32))
    b.cache.v_scale.write(np.full(b.cache.v_scale.numel, s, np.float32))
    b.v[:] = 448.0 * float(s)


@pytest.mark.parametrize("new", [1, 33])
@pytest.mark.parametrize("value,length", [(1e35, 8192), (3e38, 40), (3e38, 9000), (1e-30, 9000)])
def test_means_of_large_and_small_values(value, length, new):
    """Sums of many large values may pass f32 where their mean does not: of few rows and of many, in one block and in parts."""
    b = Batch([(new, length)], 4, 1, 64, 64)
    set_values(b, value)
    b.check()
    b.q[:] = 0.0  # equal weights
    b.check()


# ------------------------------------------------------------------ scales far apart
def slots(b, i):
    """The slots of sequence i's tokens."""
    j = np.arange(b.seqs[i][1])
    return b.table[i][j // b.page] * b.page + j % b.page


def scales(b):
    """The values' scales, [slot][head]."""
    return b.cache.v_scale.read()[:b.pages * b.heads[1] * b.page].reshape(b.pages, b.heads[1], b.page).transpose(0, 2, 1).reshape(-1, b.heads[1]).copy()


def set_scales(b, s):
    """New scales of the values, [slot][head], b.v with them."""
    old = scales(b).astype(np.float64)
    s = np.asarray(s, np.float32)
    b.cache.v_scale.write(np.ascontiguousarray(s.reshape(b.pages, b.page, -1).transpose(0, 2, 1)))
    b.v = b.v / old[..., None] * s.astype(np.float64)[..., None]


def point_at(b, i, token, logit):
    """Makes every query one that sees `token` of sequence i with that logit (in all heads) and every other token with 0."""
    d = 3
    kb, ks = b.cache.k.read().view(np.uint8).copy(), b.cache.k_scale.read()
    kb = kb[:b.pages * b.heads[1] * b.page * b.dim].reshape(b.pages, b.heads[1], b.page, b.dim)
    kb[..., d] = 0
    at = slots(b, i)[token]
    kb[at // b.page, :, at % b.page, :] = 0
    kb[at // b.page, :, at % b.page, d] = TOP
    b.cache.k.write(np.ascontiguousarray(kb).reshape(-1).view(np.float32))
    b.k[..., d] = 0.0
    b.k[at] = 0.0
    b.k[at, :, d] = 448.0 * ks[:b.pages * b.heads[1] * b.page].reshape(b.pages, b.heads[1], b.page)[at // b.page, :, at % b.page].astype(np.float64)
    b.q[:] = 0.0
    b.scale = 1.0
    group = b.heads[0] // b.heads[1]
    for h in range(b.heads[0]):
        b.q[:, h, d] = np.float32(logit / b.k[at, h // group, d])


def close(b, got=None):
    """Every row against 64 bits.  A logit's error is that of its own terms, and a weight is off by 2^-40 of the largest that
    the row sees (few rows) or 2^-32 (many: scales within 2^8 share a unit), times a byte of at most 448; the sums' roundings as in
    attention_ref.py.  No term has the largest value among tokens without weight."""
    o, l = b.run() if got is None else got
    s = scales(b).astype(np.float64)
    group = b.heads[0] // b.heads[1]
    for i, (n, length) in enumerate(b.seqs):
        at, j = slots(b, i), np.arange(length)
        for t in range(n):
            p = length - n + t
            seen = (j <= p) & ((j > p - b.window) if b.window else True)
            for h in range(b.heads[0]):
                row, kh = b.start[i] + t, h // group
                k, v, sc, q = b.k[at[seen], kh], b.v[at[seen], kh], s[at[seen], kh], b.q[row, h].astype(np.float64)
                x = k @ q * b.scale
                ds = (b.dim / 8 + 12) * 2 * U * (np.abs(k) @ np.abs(q)) * b.scale
                e = np.exp(x - x.max())
                total = e.sum()
                want = e @ v / total
                add = (2 * 64 + len(j) / 128 + 40) * 2 * U
                tol = (np.abs(v).T @ (e * (ds + add)) + np.abs(want) * (e @ ds)) / total + 2.0 ** -32 * 448 * len(v) * (e * sc).max() / total
                assert np.all(np.abs(o[row, h] - want) <= tol), (i, t, h, np.abs(o[row, h] - want).max(), np.abs(want).max(), tol.max())
                assert abs(l[row, h] - x.max() - np.log(total)) <= (e @ ds) / total + add + 2 * U * abs(x.max() + np.log(total))


FORMS = [(1, 100, 4), (2, 100, 4), (2, 300, 12), (20, 100, 4), (33, 40, 4), (70, 400, 12)]  # new, length, query heads of the kv head


@pytest.mark.parametrize("shift", [9, 24, 45, 100])
@pytest.mark.parametrize("group", [4, 12])
def test_a_row_does_not_see_the_next_token(group, shift):
    """Two new tokens, the second one's value 2^shift times the first's: the first row is bit for bit what it is without."""
    b = Batch([(2, 2)], group, 1, 64, 16)
    s = scales(b)
    s[slots(b, 0)] = 0.01
    set_scales(b, s)
    o, l = b.run()
    s[slots(b, 0)[1]] *= np.float32(2.0) ** shift
    set_scales(b, s)
    got = b.run()
    assert np.array_equal(got[0][0].view(np.uint32), o[0].view(np.uint32)) and np.array_equal(got[1][0], l[0])
    close(b, got)


@pytest.mark.parametrize("shift", [9, 24, 45, 100])
@pytest.mark.parametrize("new,length,group", [f for f in FORMS if f[0] > 1])
def test_rows_do_not_see_values_behind_them(new, length, group, shift):
    """The last token's value is 2^shift times another: rows before it are bit for bit what they are without.  Tiles of many rows
    take tokens of scales within 2^8 together, so where others are that near to the large one the sums' order and the unit differ,
    and with them roundings: then both results are held to the bounds against 64 bits alone."""
    b = Batch([(new, length)], group, 1, 64, 16)
    s = scales(b)
    s[slots(b, 0)[-1]] = s[slots(b, 0)[0]]
    set_scales(b, s)
    o, l = b.run()
    close(b, (o, l))
    s[slots(b, 0)[-1]] *= np.float32(2.0) ** shift
    set_scales(b, s)
    got = b.run()
    if new * group <= 16 or s[slots(b, 0)].max() > 2.0 ** 8 * np.sort(s[slots(b, 0), 0])[-2]:
        assert np.array_equal(got[0][:-1].view(np.uint32), o[:-1].view(np.uint32)) and np.array_equal(got[1], l)
    close(b, got)


@pytest.mark.parametrize("shift", [12, 24, 45, 100])
@pytest.mark.parametrize("new,length,group", FORMS)
def test_a_large_value_without_weight(new, length, group, shift):
    """A token that every row sees, of no weight, with a value 2^shift times the others': they keep their bits."""
    b = Batch([(new, length)], group, 1, 64, 16)
    point_at(b, 0, 5, -200.0)
    s = scales(b)
    s[slots(b, 0)[5]] *= np.float32(2.0) ** shift
    set_scales(b, s)
    close(b)


@pytest.mark.parametrize("zero", ["bytes", "smallest scale", "scale"])
@pytest.mark.parametrize("logit", [14.0, 21.0, 35.0])
@pytest.mark.parametrize("new,length,group", FORMS)
def test_all_weight_on_a_token_without_value(new, length, group, logit, zero):
    """One token takes all but 2^-20 .. 2^-50 of the weight and has no value: what the others bring keeps f32's bits, in its tile and
    in others."""
    b = Batch([(new, length)], group, 1, 64, 16)
    point_at(b, 0, 5, logit)
    at = slots(b, 0)[5]
    s = scales(b)
    if zero == "bytes":  # (of the scale of a row that a token of like size has)
        s[at] = s.min() / 64
        vb = b.cache.v.read().view(np.uint8).copy()
        vb.reshape(b.pages, 1, b.page, -1)[at // b.page, :, at % b.page] = 0
        b.cache.v.write(vb.view(np.float32))
        b.v[at] = 0.0
    set_scales(b, s)
    if zero != "bytes":
        s[at] = np.float32(2.0 ** -100 / 448) if zero == "smallest scale" else 0.0
        b.v[at] = 0.0 if zero == "scale" else b.v[at] / scales(b)[at].astype(np.float64)[..., None] * s[at].astype(np.float64)[..., None]
        b.cache.v_scale.write(np.ascontiguousarray(s.reshape(b.pages, b.page, -1).transpose(0, 2, 1)))
    o, l = b.run()
    # of the token itself: its scale's share of the bound
    close(b, (o, l))


@pytest.mark.parametrize("window", [0, 30])
@pytest.mark.parametrize("low,high", [(-60, 21), (-100, 118), (0, 9)])
@pytest.mark.parametrize("new,length,group", FORMS)
def test_scales_over_many_powers_of_two(new, length, group, low, high, window):
    b = Batch([(new, length), (1, 60)], group, 1, 64, 16, window=window)
    g = np.random.default_rng([0x5C, new, length, group, 200 + low])
    set_scales(b, np.float32(2.0) ** g.integers(low, high, scales(b).shape).astype(np.float32) * np.float32(1.3))
    close(b)


def test_sums_stay_short_where_pages_are_missing():
    """A single token over 8.5 million, of which every block's warps miss each sixteenth group of 16 tokens (twelve warps take groups
    in turn, blocks have equal shares in units of 128 tokens): the sums between two flushes are no longer for it.  All logits are
    zero and the values 448 and 13 of a unit in turn, so that the mean is half their sum and no sum is exact."""
    d, page, dim, blocks, warps = device(), 16, 16, 148, 12
    units = blocks * 450
    pages = units * 128 // page
    c = d.kv_cache(pages, 1, dim, page)
    value = np.float32(0.7123457)
    c.v.write(np.tile(np.repeat(np.uint8([TOP, 0x55]), dim), c.v.numel * 4 // (2 * dim)).view(np.float32))
    c.v_scale.write(np.full(c.v_scale.numel, value, np.float32))
    c.k_scale.write(np.ones(c.k_scale.numel, np.float32))
    table = np.arange(pages)
    begin = (units * np.arange(blocks + 1) // blocks) * 8  # of each block, in groups
    at = table - begin[np.searchsorted(begin, table, side="right") - 1]
    table[at // warps % 16 == 15] = -1
    out, lse = blank(1, dim), blank(1, 1)
    d.attention_paged(c, 1, 1, out, up(np.ones(dim)), ints(table), ints([0, 1]), ints([pages * page]), 1, pages, max_new=1, scale=1.0, lse=lse)
    want, count = (448.0 + 13.0) / 2 * float(value), int((table >= 0).sum()) * page
    # 16 tensor instructions between flushes, each losing up to a step (2 U) of the sum; 300 / 16 flushes, 12 warps and 148 parts with a
    # rounding each; the weights' halves (4 U), and some ten roundings more
    assert np.all(np.abs(get(out, dim) - want) <= (16 * 2 + 19 + 12 + 148 + 4 + 10) * U * want)
    assert abs(get(lse, 1)[0] - np.log(count)) <= (300 * 4 + 12 + 148 + 10) * U + 4 * U * np.log(count)


@pytest.mark.parametrize("new", [1, 33])
def test_scales_near_the_end_and_queries_near_zero(new):
    """Every finite scale: the largest with queries of zero (equal weights) and with queries below the least normal value (logits of
    ordinary size)."""
    b = Batch([(new, 70)], 4, 1, 64, 16)
    q = b.q.copy()
    b.q[:] = 0.0
    for scale in (3.4e38, 1e38, 1e-45):
        b.scale = float(np.float32(scale))
        close(b)
    b.q[:] = q * np.float32(2.0) ** -126
    b.q[:, 1] = q[:, 1] * np.float32(2.0) ** -132  # (few bits are left of them)
    b.scale = float(np.float32(2.0 ** 125))
    close(b)


@pytest.mark.parametrize("new,length,group", FORMS)
def test_scales_that_are_none_stay_with_their_rows(new, length, group):
    """Scales below zero, infinite or NaN (the first two no call of the library writes): every call ends, and the rows that do not see them
    are right.  The token before the last has one, so that all rows but the last two of the sequence hold to the bounds; of a sequence
    beside it all do."""
    for bad in (-1.0, -2.0 ** 100, np.inf, np.nan, -0.0):
        b = Batch([(new, length), (new, 50 + new)], group, 1, 64, 16)
        s, v = scales(b), b.v.copy()
        at = slots(b, 0)[length - 2]
        s[at] = bad
        b.cache.v_scale.write(np.ascontiguousarray(s.reshape(b.pages, b.page, -1).transpose(0, 2, 1)))
        o, l = b.run()
        keep = np.ones(b.rows, bool)
        keep[max(0, new - 2):new] = False
        s[at], b.v = 1.0, v
        b.cache.v_scale.write(np.ascontiguousarray(s.reshape(b.pages, b.page, -1).transpose(0, 2, 1)))
        want = [b.want(i) for i in range(2)]
        out, lse, tol, ltol = (np.concatenate([w[k] for w in want]) for k in range(4))
        assert np.all(np.abs(o - out)[keep] <= tol[keep]) and np.all(np.abs(l - lse)[keep] <= ltol[keep])


@pytest.mark.parametrize("dim", [16, 64, 96, 128])
@pytest.mark.parametrize("seqs", [[(40, 40), (150, 333)], [(30, 9001)], [(1, 300), (90, 700), (3, 40)]])
def test_rows_that_are_not_aligned(dim, seqs):
    """Queries and outputs at strides that are no multiple of 16 bytes."""
    Batch(seqs, 10, 2, dim, 32, extra=3).check()
    Batch(seqs, 10, 2, dim, 32, extra=4).check()
