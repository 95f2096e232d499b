"""Language-model row operators without a GPU: operand layout, the e4m3 values, and the refusals.

Entry points check their arguments before they touch the device, so a refused call needs none: the
device handle here is a block of zeros that no refused call may read."""
import ctypes as C

import numpy as np
import pytest

import mag_b200 as MB

L = MB.load_library()
FAKE = C.create_string_buffer(C.sizeof(MB.ComputeDevice))
DEV = C.addressof(FAKE)
BIG = 1 << 31


def test_operand_layout():
    for cols, ld in ((1, 128), (127, 128), (128, 128), (129, 256), (5000, 5120)):
        assert L.mag_cuda_e4m3_ld(cols) == MB.e4m3_ld(cols) == ld
    assert L.mag_cuda_e4m3_ld(0) == 0 and L.mag_cuda_e4m3_ld(-5) == 0 and L.mag_cuda_e4m3_ld((1 << 63) - 1) == 0
    assert L.mag_cuda_e4m3_scales(5, 300, MB.E4M3_ROW) == 15
    assert L.mag_cuda_e4m3_scales(129, 300, MB.E4M3_BLOCK) == 6
    assert L.mag_cuda_e4m3_scales(5, 300, 2) == 0 and L.mag_cuda_e4m3_scales(-1, 300, 0) == 0


def test_e4m3_values():
    v = MB.e4m3_values()
    assert v[0x7E] == 448.0 and v[0xFE] == -448.0 and v[0x08] == 2.0 ** -6 and v[0x01] == 2.0 ** -9
    assert np.isnan(v[0x7F]) and np.isnan(v[0xFF]) and v[0x38] == 1.0
    finite = v[:0x7F]
    assert np.all(np.diff(finite) > 0)


A, B16, B32 = 0x1000, 0x2010, 0x3020  # well aligned addresses that no refused call reads


def refused(name, good, changes):
    """The good call's arguments with one change each: all refused."""
    fn = getattr(L, name)
    for at, value in changes:
        args = list(good)
        args[at] = value
        assert fn(*args) == MB.E_INVALID, (name, at, value)


def test_quantize_refusals():
    good = (DEV, A, B16, B32, 4, 8, 0, 0)
    refused("mag_cuda_quantize_e4m3", good, [(0, None), (1, None), (2, None), (3, None), (1, A + 8), (2, B16 + 2),
                                             (3, B32 + 1), (4, -1), (4, BIG), (5, 0), (5, -3), (5, BIG), (6, 2), (6, -1)])
    assert L.mag_cuda_quantize_e4m3(DEV, A, B16, B32, 0, 8, 0, 0) == 0


def test_matmul_refusals():
    good = (DEV, A, A, B16, B32, A, 4, 8, 4, 1)
    refused("mag_cuda_matmul_e4m3", good, [(i, None) for i in range(6)] + [
        (1, A + 2), (2, A + 4), (3, B16 + 1), (4, B32 + 8), (5, A + 3), (6, -1), (6, BIG), (7, 0), (7, -1), (7, BIG),
        (8, -1), (8, BIG), (9, 2), (9, -1)])
    assert L.mag_cuda_matmul_e4m3(DEV, A, A, B16, B32, A, BIG - 300, 8, BIG - 300, 1) == MB.E_INVALID
    assert L.mag_cuda_matmul_e4m3(DEV, A, A, B16, B32, A, 0, 8, 4, 1) == 0
    assert L.mag_cuda_matmul_e4m3(DEV, A, A, B16, B32, A, 4, 8, 0, 1) == 0


def test_rmsnorm_refusals():
    nan, inf = float("nan"), float("inf")
    good = (DEV, A, B16, B32, 0x4000, A, 0x5000, 0x6000, 0x7000, 1e-6, 4, 8)
    refused("mag_cuda_rmsnorm_rows_f32", good, [
        (0, None), (2, None), (3, None), (6, None), (8, None), (4, A), (1, A + 2), (2, B16 + 4), (3, B32 + 1),
        (4, 0x4002), (5, A + 1), (6, 0x5001), (7, 0x6002), (8, 0x7003), (9, -1e-6), (9, nan), (9, inf), (10, -1),
        (10, BIG), (11, 0), (11, BIG)])
    assert L.mag_cuda_rmsnorm_rows_f32(DEV, None, None, None, None, None, A, None, A, 1e-6, 4, 8) == MB.E_INVALID
    assert L.mag_cuda_rmsnorm_rows_f32(*good[:10], 0, 8) == 0


def test_rmsnorm_backward_refusals():
    good = (DEV, A, A, A, A, A, A, A, 4, 8)
    refused("mag_cuda_rmsnorm_rows_backward_f32", good, [(i, None) for i in (0, 1, 3, 4, 5, 6)] +
            [(i, A + 2) for i in range(1, 8)] + [(8, -1), (8, BIG), (9, 0), (9, BIG)])
    assert L.mag_cuda_rmsnorm_rows_backward_f32(DEV, A, None, A, A, A, A, None, 0, 8) == 0


def test_logprobs_refusals():
    good = (DEV, A, A, A, A, A, A, A, 4, 8, 8, 3)
    refused("mag_cuda_token_logprobs_f32", good, [(0, None), (6, None), (7, None)] + [(i, A + 2) for i in range(1, 8)] + [
        (8, -1), (8, BIG), (9, 0), (9, BIG), (10, 7), (10, BIG), (11, -1), (11, 9), (11, 33)])
    nothing = (DEV, None, None, None, None, None, A, A, 4, 8, 8)
    assert L.mag_cuda_token_logprobs_f32(*nothing, 3) == MB.E_INVALID
    assert L.mag_cuda_token_logprobs_f32(*nothing, 0) == MB.E_INVALID
    assert L.mag_cuda_token_logprobs_f32(*good[:8], 0, 8, 8, 3) == 0


def test_logprobs_backward_refusals():
    X = 0x9000
    good = (DEV, A, X, A, A, A, A, A, 4, 8, 8, 8)
    refused("mag_cuda_token_logprobs_backward_f32", good, [(i, None) for i in (0, 1, 2, 3, 4, 5)] +
            [(i, A + 2) for i in range(1, 8)] + [(8, -1), (8, BIG), (9, 0), (10, 7), (11, 7), (10, BIG), (11, BIG)])
    assert L.mag_cuda_token_logprobs_backward_f32(DEV, A, X, A, A, A, None, None, 4, 8, 8, 8) == MB.E_INVALID
    assert L.mag_cuda_token_logprobs_backward_f32(DEV, X, X, A, A, A, A, A, 4, 8, 8, 9) == MB.E_INVALID
    assert L.mag_cuda_token_logprobs_backward_f32(*good[:8], 0, 8, 8, 8) == 0


def test_python_refusals_raise():
    d = MB.Device.__new__(MB.Device)  # the methods' own checks come from the library
    d.L, d.p, d.alive = L, DEV, False
    with pytest.raises(MB.CudaError):
        d.quantize_e4m3(4, 0, A, A, A)
    with pytest.raises(MB.CudaError):
        d.token_logprobs(4, 8, A, top=40, top_id=A)
    for rows, cols in ((0, 5), (5, 0)):
        with pytest.raises(ValueError):
            d.e4m3(rows, cols)
