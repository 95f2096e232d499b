/*
 * lm_rows.c - entry points of the language-model row operators (host side, C): argument checks,
 * buffer bookkeeping and launch of the norm, the e4m3 quantiser and product, and the token log
 * probabilities.  Nothing of the device is touched before the arguments have been checked.
 */
#include "magnetron_cuda.h"
#include "mcu_device.h"
#include "mcu_kernels.h"
#include "mcu_args.h"

#include <math.h>

int64_t mag_cuda_e4m3_ld(int64_t cols) { return cols > 0 && cols < MCU_MAX_DIM ? (cols + 127) / 128 * 128 : 0; }

int64_t mag_cuda_e4m3_scales(int64_t rows, int64_t cols, int group) {
    if (rows <= 0 || rows >= MCU_MAX_DIM || cols <= 0 || cols >= MCU_MAX_DIM || (group != MAG_CUDA_E4M3_ROW && group != MAG_CUDA_E4M3_BLOCK)) return 0;
    return (group == MAG_CUDA_E4M3_BLOCK ? (rows + 127) / 128 : rows) * (mag_cuda_e4m3_ld(cols) / 128);
}

int mag_cuda_quantize_e4m3(mag_compute_device_t* dvc, uint8_t* q, float* s, const float* x, int64_t rows, int64_t cols,
                           int group, int transpose) {
    if (!dvc || !q || !s || !x || bad_matrix(rows, cols) || odd16(q) || odd4(s) || odd4(x) ||
        (group != MAG_CUDA_E4M3_ROW && group != MAG_CUDA_E4M3_BLOCK))
        return MAG_CUDA_E_INVALID;
    if (!rows) return 0;
    const int64_t a = transpose ? cols : rows, b = transpose ? rows : cols;
    const mcu_buf bufs[] = {{x, 0, 0},
                            {q, (size_t)(a * mag_cuda_e4m3_ld(b)), 1},
                            {s, (size_t)mag_cuda_e4m3_scales(a, b, group) * 4, 1}};
    mcu_call c;
    int k = 0, rc = mcu_call_begin(&c, dvc, bufs, 3, 0);
    if (rc) return rc;
    rc = mcu_launch_quantize_e4m3(q, s, x, rows, cols, group == MAG_CUDA_E4M3_BLOCK, transpose != 0, c.stream, &k);
    return mcu_call_end(&c, rc, k);
}

int mag_cuda_matmul_e4m3(mag_compute_device_t* dvc, float* r, const uint8_t* xq, const float* xs, const uint8_t* yq,
                         const float* ys, int64_t M, int64_t K, int64_t N, int y_group) {
    if (!dvc || !r || !xq || !xs || !yq || !ys || bad_matrix(M, K) || bad_matrix(N, K) || M * N > ((int64_t)1 << 42) || odd4(r) || odd4(xs) ||
        odd4(ys) || odd16(xq) || odd16(yq) || (y_group != MAG_CUDA_E4M3_ROW && y_group != MAG_CUDA_E4M3_BLOCK))
        return MAG_CUDA_E_INVALID;
    if (!M || !N) return 0;
    const mcu_buf bufs[] = {{xq, 0, 0}, {xs, 0, 0}, {yq, 0, 0}, {ys, 0, 0}, {r, (size_t)(M * N) * 4, 1}};
    mcu_call c;
    int k = 0, rc = mcu_call_begin(&c, dvc, bufs, 5, 0);
    if (rc) return rc;
    rc = mcu_launch_matmul_e4m3(r, xq, xs, yq, ys, M, K, N, y_group == MAG_CUDA_E4M3_BLOCK, c.status, c.stream, &k);
    return mcu_call_end(&c, rc, k);
}

int mag_cuda_rmsnorm_rows_f32(mag_compute_device_t* dvc, float* y, uint8_t* q, float* s, float* h, float* rstd,
                              const float* x, const float* residual, const float* w, float eps, int64_t rows,
                              int64_t cols) {
    if (!dvc || (!y && !q) || !q != !s || !x || !w || bad_matrix(rows, cols) || !(eps >= 0.0f) || isinf(eps) ||
        odd4(y) || odd16(q) || odd4(s) || odd4(h) || odd4(rstd) || odd4(x) || odd4(residual) || odd4(w) || (h && h == y))
        return MAG_CUDA_E_INVALID;
    if (!rows) return 0;
    const size_t n = (size_t)(rows * cols) * 4;
    const mcu_buf bufs[] = {{x, 0, 0}, {residual, 0, 0}, {w, 0, 0}, {y, n, 1}, {h, n, 1}, {rstd, (size_t)rows * 4, 1},
                            {q, (size_t)(rows * mag_cuda_e4m3_ld(cols)), 1},
                            {s, (size_t)mag_cuda_e4m3_scales(rows, cols, MAG_CUDA_E4M3_ROW) * 4, 1}};
    mcu_call c;
    int k = 0, rc = mcu_call_begin(&c, dvc, bufs, 8, 0);
    if (rc) return rc;
    rc = mcu_launch_rmsnorm(y, q, s, h, rstd, x, residual, w, eps, rows, cols, c.stream, &k);
    return mcu_call_end(&c, rc, k);
}

int mag_cuda_rmsnorm_rows_backward_f32(mag_compute_device_t* dvc, float* dx, float* dw, const float* dy,
                                       const float* h, const float* w, const float* rstd, const float* dh,
                                       int64_t rows, int64_t cols) {
    if (!dvc || !dx || !dy || !h || !w || !rstd || bad_matrix(rows, cols) || odd4(dx) || odd4(dw) || odd4(dy) ||
        odd4(h) || odd4(w) || odd4(rstd) || odd4(dh))
        return MAG_CUDA_E_INVALID;
    const mcu_buf bufs[] = {{dy, 0, 0}, {h, 0, 0}, {w, 0, 0}, {rstd, 0, 0}, {dh, 0, 0},
                            {dx, (size_t)(rows * cols) * 4, 1}, {dw, (size_t)cols * 4, 1}};
    mcu_call c;
    int k = 0, rc;
    if (!rows) {
        if (!dw) return 0;
        if ((rc = mcu_call_begin(&c, dvc, bufs + 6, 1, 0))) return rc;
        return mcu_call_end(&c, (int)cudaMemsetAsync(dw, 0, (size_t)cols * 4, c.stream), 0);
    }
    rc = mcu_call_begin(&c, dvc, bufs, 7, dw ? mcu_rmsnorm_backward_scratch_bytes(rows, cols) : 0);
    if (rc) return rc;
    rc = mcu_launch_rmsnorm_backward(dx, dw, dy, h, w, rstd, dh, rows, cols, c.scratch, c.status, c.stream, &k);
    return mcu_call_end(&c, rc, k);
}

int mag_cuda_token_logprobs_f32(mag_compute_device_t* dvc, float* logp, float* lse, float* entropy, float* top_logp,
                                int32_t* top_id, const float* x, const int32_t* id, int64_t rows, int64_t cols,
                                int64_t x_s1, int top) {
    if (!dvc || !x || bad_matrix(rows, cols) || x_s1 < cols || x_s1 >= MCU_MAX_DIM || top < 0 || top > MAG_CUDA_TOP_MAX ||
        top > cols || (logp && !id) || odd4(logp) || odd4(lse) || odd4(entropy) || odd4(top_logp) || odd4(top_id) ||
        odd4(x) || odd4(id) || (!logp && !lse && !entropy && (!top || (!top_logp && !top_id))))
        return MAG_CUDA_E_INVALID;
    if (!rows) return 0;
    if (!top) top_logp = NULL, top_id = NULL;
    if (!top_logp && !top_id) top = 0;
    const size_t n = (size_t)rows * 4;
    const mcu_buf bufs[] = {{x, 0, 0}, {id, 0, 0}, {logp, n, 1}, {lse, n, 1}, {entropy, n, 1}, {top_logp, n * (size_t)top, 1},
                            {top_id, n * (size_t)top, 1}};
    mcu_call c;
    int k = 0, rc = mcu_call_begin(&c, dvc, bufs, 7, 0);
    if (rc) return rc;
    rc = mcu_launch_logprobs(logp, lse, entropy, top_logp, top_id, x, id, rows, cols, x_s1, top, c.stream, &k);
    return mcu_call_end(&c, rc, k);
}

int mag_cuda_token_logprobs_backward_f32(mag_compute_device_t* dvc, float* dx, const float* x, const int32_t* id,
                                         const float* lse, const float* entropy, const float* g_logp,
                                         const float* g_entropy, int64_t rows, int64_t cols, int64_t x_s1,
                                         int64_t dx_s1) {
    if (!dvc || !dx || !x || !lse || (!g_logp && !g_entropy) || (g_logp && !id) || (g_entropy && !entropy) ||
        bad_matrix(rows, cols) || x_s1 < cols || dx_s1 < cols || x_s1 >= MCU_MAX_DIM || dx_s1 >= MCU_MAX_DIM ||
        (dx == x && x_s1 != dx_s1) || odd4(dx) || odd4(x) || odd4(id) || odd4(lse) || odd4(entropy) || odd4(g_logp) ||
        odd4(g_entropy))
        return MAG_CUDA_E_INVALID;
    if (!rows) return 0;
    /* rows of padded width are written in part: the padding keeps what it holds */
    const mcu_buf bufs[] = {{x, 0, 0}, {id, 0, 0}, {lse, 0, 0}, {entropy, 0, 0}, {g_logp, 0, 0}, {g_entropy, 0, 0},
                            {dx, dx_s1 == cols ? (size_t)(rows * cols) * 4 : 4, 1}};
    mcu_call c;
    int k = 0, rc = mcu_call_begin(&c, dvc, bufs, 7, 0);
    if (rc) return rc;
    rc = mcu_launch_logprobs_backward(dx, x, id, lse, entropy, g_logp, g_entropy, rows, cols, x_s1, dx_s1, c.stream, &k);
    return mcu_call_end(&c, rc, k);
}
