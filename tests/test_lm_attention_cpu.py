"""Attention operators without a GPU: the rotation's table and the refusals.

Entry points check their arguments before they touch the device, so a refused call needs none: the
device handle here is a block of zeros that no refused call may read."""
import ctypes as C
import math

import numpy as np
import pytest

import mag_b200 as MB

L = MB.load_library()
FAKE = C.create_string_buffer(C.sizeof(MB.ComputeDevice))
DEV = C.addressof(FAKE)
BIG = 1 << 31
A, B, D = 0x1000, 0x2010, 0x3020  # well aligned addresses that no refused call reads
NAN, INF = math.nan, math.inf


def refused(name, good, changes):
    """The good call's arguments with one change each: all refused."""
    fn = getattr(L, name)
    for at, value in changes:
        args = list(good)
        args[at] = value
        assert fn(*args) == MB.E_INVALID, (name, at, value)


def cache(**kw):
    f = {"k": A, "v": B, "k_scale": D, "v_scale": A, "pages": 4, "heads": 2, "head_dim": 64, "page_size": 16}
    f.update(kw)
    c = MB.KvCacheStruct(*(f[n] for n, _ in MB.KvCacheStruct._fields_))
    KEEP.append(c)
    return C.addressof(c)


def rotation(**kw):
    f = {"pos": A, "inv_freq": B, "rot": 16, "interleaved": 0, "magnitude": 1.0}
    f.update(kw)
    c = MB.RotationStruct(*(f[n] for n, _ in MB.RotationStruct._fields_))
    KEEP.append(c)
    return C.addressof(c)


KEEP = []
BAD_CACHES = [{"k": None}, {"v": None}, {"k_scale": None}, {"v_scale": None}, {"k": A + 8}, {"v": A + 1}, {"k_scale": A + 4},
              {"v_scale": A + 8}, {"pages": 0}, {"pages": -1}, {"heads": 0}, {"heads": 65536}, {"head_dim": 8}, {"head_dim": 136},
              {"head_dim": 100}, {"head_dim": 0}, {"page_size": 8}, {"page_size": 24}, {"page_size": 2048}, {"page_size": 0},
              {"pages": 1 << 27}, {"pages": (1 << 27) - 1, "heads": 2000}]
BAD_ROTATIONS = [{"rot": -8}, {"rot": 4}, {"rot": 72}, {"pos": None}, {"inv_freq": None}, {"pos": A + 2}, {"inv_freq": A + 1},
                 {"magnitude": NAN}, {"magnitude": INF}]


def test_rotate_heads_refusals():
    name = "mag_cuda_rotate_heads_f32"
    good = (DEV, A, B, D, A, 1e-6, rotation(), 4, 2, 64, 128, 128)
    refused(name, good, [(0, None), (1, None), (3, None), (4, None), (1, A + 2), (2, A + 1), (3, A + 3), (4, B + 2), (5, -1.0), (5, NAN),
                         (5, INF), (7, -1), (7, BIG), (8, 0), (8, 65536), (9, 0), (9, 4), (9, 68), (9, 264), (10, 127), (10, BIG),
                         (11, 127), (11, BIG)] + [(6, rotation(**r)) for r in BAD_ROTATIONS])
    refused(name, (DEV, A, None, A, None, 1e-6, None, 4, 2, 64, 128, 128), [(11, 256)])  # in place, other strides
    assert getattr(L, name)(DEV, A, None, D, None, 1e-6, rotation(rot=0, pos=None, inv_freq=None, magnitude=NAN), 0, 2, 64, 128, 128) == 0


def test_rotate_heads_backward_refusals():
    name = "mag_cuda_rotate_heads_backward_f32"
    good = (DEV, A, B, D, A, B, D, rotation(), 4, 2, 64, 128, 128, 128)
    refused(name, good, [(0, None), (1, None), (3, None), (4, None), (5, None), (6, None), (1, A + 2), (2, A + 1), (3, A + 3), (4, B + 2),
                         (5, B + 1), (6, B + 2), (8, -1), (8, BIG), (9, 0), (10, 12), (11, 127), (12, 100), (13, 5), (11, BIG)] +
            [(7, rotation(**r)) for r in BAD_ROTATIONS])
    plain = (DEV, A, None, D, None, None, None, None, 4, 2, 64, 128, 128, 0)
    refused(name, plain, [(2, B), (4, B), (6, B)])
    refused(name, (DEV, A, None, A, B, B, D, None, 4, 2, 64, 128, 128, 128), [(11, 256), (12, 256)])
    refused(name, (DEV, A, None, D, A, B, D, None, 4, 2, 64, 128, 128, 128), [(11, 256), (13, 256)])
    assert getattr(L, name)(DEV, A, None, D, None, None, None, None, 0, 2, 64, 128, 128, 0) == 0


def test_kv_write_refusals():
    name = "mag_cuda_kv_write"
    good = (DEV, cache(), A, B, D, A, B, D, A, 1e-6, rotation(), 4, 6, 128, 128, 384, 384)
    refused(name, good, [(0, None), (1, None), (2, None), (3, None), (4, None), (6, None), (7, None), (2, A + 2), (3, A + 1), (4, A + 2),
                         (5, A + 3), (6, A + 1), (7, A + 2), (8, A + 2), (9, NAN), (9, -1.0), (11, -1), (11, BIG), (12, 0), (12, 65536),
                         (13, 127), (14, 127), (15, 383), (16, 383), (13, BIG), (15, BIG)] +
            [(1, cache(**c)) for c in BAD_CACHES] + [(10, rotation(**r)) for r in BAD_ROTATIONS])
    refused(name, (DEV, cache(), A, B, D, A, None, None, None, 1e-6, None, 4, 0, 128, 128, 0, 0), [(8, A)])  # a weight without queries
    refused(name, (DEV, cache(), A, B, D, A, B, B, None, 1e-6, None, 4, 6, 128, 128, 384, 384), [(15, 400), (16, 400)])
    assert getattr(L, name)(DEV, cache(), A, B, D, A, None, None, None, 1e-6, None, 0, 0, 128, 128, 0, 0) == 0


def test_kv_read_refusals():
    name = "mag_cuda_kv_read"
    good = (DEV, cache(), A, B, D, 4, 128, 128)
    refused(name, good, [(0, None), (1, None), (4, None), (2, B), (2, A + 2), (3, B + 2), (4, D + 1), (5, -1), (5, BIG), (6, 127), (7, 127)] +
            [(1, cache(**c)) for c in BAD_CACHES])
    assert getattr(L, name)(DEV, cache(), None, None, D, 4, 128, 128) == MB.E_INVALID
    assert getattr(L, name)(DEV, cache(), A, None, D, 0, 128, 0) == 0


def test_attention_refusals():
    name = "mag_cuda_attention_paged_f32"
    good = (DEV, A, B, D, cache(), A, B, D, 2, 8, 5, 3, 6, 0.125, 0, 384, 384)
    refused(name, good, [(0, None), (1, None), (3, None), (4, None), (5, None), (6, None), (7, None), (1, A + 2), (2, B + 1), (3, D + 2),
                         (5, A + 1), (6, A + 2), (7, A + 3), (8, -1), (8, BIG), (9, 0), (9, BIG), (9, 1 << 27), (10, -1), (10, BIG),
                         (11, -1), (11, BIG), (12, 0), (12, -2), (12, 5), (12, 65536), (13, NAN), (13, -0.5), (13, INF), (14, -1), (15, 383),
                         (16, 383), (15, BIG), (1, D)] + [(4, cache(**c)) for c in BAD_CACHES])
    for at in (8, 10, 11):
        args = list(good)
        args[at] = 0
        assert getattr(L, name)(*args) == 0


def test_cache_sizes_are_checked_before_storage_is_taken():
    class Never(MB.Device):
        def __init__(self):
            self.alive = False

    for pages, heads, dim, page in ((0, 2, 64, 16), (4, 0, 64, 16), (4, 2, 60, 16), (4, 2, 144, 16), (4, 2, 64, 8), (4, 2, 64, 48)):
        with pytest.raises(ValueError):
            Never().kv_cache(pages, heads, dim, page)


def test_rope_frequencies():
    f = MB.rope_frequencies(128, 10000.0)
    assert f.dtype == np.float32 and f.shape == (64,) and f[0] == 1.0
    assert np.allclose(f[1:] / f[:-1], 10000.0 ** (-2.0 / 128), rtol=1e-6)
    assert np.allclose(MB.rope_frequencies(128, 10000.0, factor=4.0), f / 4.0, rtol=1e-6)
    g = MB.rope_frequencies(128, 10000.0, factor=4.0, original=4096, low=1.0, high=32.0)
    turns = 4096 * f.astype(np.float64) / (2 * np.pi)
    assert np.array_equal(g[turns >= 32.1], f[turns >= 32.1])          # fast pairs keep their frequency
    assert np.allclose(g[turns <= 0.99], f[turns <= 0.99] / 4.0)       # slow ones take the whole factor
    between = (turns > 1.01) & (turns < 31.9)
    assert between.any() and np.all(g[between] < f[between]) and np.all(g[between] > f[between] / 4.0)
    assert MB.rope_frequencies(0).shape == (0,)
    for bad in ({"rot": 7}, {"rot": 8, "base": 0.0}, {"rot": 8, "factor": -1.0}, {"rot": 8, "low": 4.0, "high": 4.0}):
        with pytest.raises(ValueError):
            MB.rope_frequencies(**bad)
