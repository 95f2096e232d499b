// k_rmsnorm.cu - root-mean-square norm of rows with the residual's addition, f32 and e4m3 outputs, and
// its gradient (mag_cuda_rmsnorm_rows_f32, mag_cuda_rmsnorm_rows_backward_f32).
#include <cuda_runtime.h>
#include <cstdint>
#include "mcu_kernels.h"
#include "mcu_lm.cuh"

using namespace mcu;

namespace {

constexpr int kThreads = 256;

// Sum over the block of 256, the same on every thread.
__device__ float block_sum(float v) {
    __shared__ float sh[kThreads / 32];
    v = warp_sum_f(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = 0.0f;
    for (int i = 0; i < kThreads / 32; ++i) t += sh[i];
    return t;
}

// One block per row, two passes over it.
__global__ void __launch_bounds__(kThreads) rmsnorm_row(float* y, uint8_t* q, float* s, float* h, float* rstd,
                                                        const float* x, const float* res, const float* w, float eps,
                                                        int64_t cols) {
    const int64_t row = blockIdx.x, o = row * cols;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float a = 0.0f;
    for (int64_t c = threadIdx.x; c < cols; c += kThreads) {
        const float v = res ? x[o + c] + res[o + c] : x[o + c];
        a += v * v;
    }
    const float root = rsqrtf(block_sum(a) / (float)cols + eps);
    if (rstd && threadIdx.x == 0) rstd[row] = root;
    const int64_t groups = (cols + 127) / 128;
    for (int64_t g = warp; g < groups; g += kThreads / 32) {
        float v[4];
        uint32_t top = 0;
        for (int i = 0; i < 4; ++i) {
            const int64_t c = g * 128 + lane * 4 + i;
            v[i] = 0.0f;
            if (c < cols) {
                const float t = res ? x[o + c] + res[o + c] : x[o + c];
                if (h) h[o + c] = t;
                v[i] = t * root * w[c];
                if (y) y[o + c] = v[i];
            }
            top = max(top, abs_bits(v[i]));
        }
        if (q) {
            const float sc = e4m3_scale(__reduce_max_sync(0xffffffffu, top)), inv = __frcp_rn(sc);
            if (lane == 0) s[row * groups + g] = sc;
            *(uint32_t*)(q + (row * groups + g) * 128 + lane * 4) = e4m3x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
        }
    }
}

__global__ void __launch_bounds__(kThreads) rmsnorm_backward_row(float* dx, const float* dy, const float* h,
                                                                 const float* w, const float* rstd, const float* dh,
                                                                 int64_t cols) {
    const int64_t row = blockIdx.x, o = row * cols;
    float a = 0.0f;
    for (int64_t c = threadIdx.x; c < cols; c += kThreads) a += dy[o + c] * w[c] * h[o + c];
    const float root = rstd[row], f = root * root * (block_sum(a) / (float)cols);
    for (int64_t c = threadIdx.x; c < cols; c += kThreads) {
        const float u = root * (dy[o + c] * w[c] - h[o + c] * f);
        dx[o + c] = dh ? dh[o + c] + u : u;
    }
}

__global__ void __launch_bounds__(kThreads) rmsnorm_backward_weight(float* dw, const float* dy, const float* h,
                                                                    const float* rstd, int64_t rows, int64_t cols) {
    const int64_t c = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (c >= cols) return;
    float a = 0.0f;
    for (int64_t r = 0; r < rows; ++r) a += dy[r * cols + c] * (h[r * cols + c] * rstd[r]);
    dw[c] = a;
}

}  // namespace

extern "C" int mcu_launch_rmsnorm(float* y, uint8_t* q, float* s, float* h, float* rstd, const float* x,
                                  const float* res, const float* w, float eps, int64_t rows, int64_t cols,
                                  cudaStream_t st, int* launches) {
    rmsnorm_row<<<(unsigned)rows, kThreads, 0, st>>>(y, q, s, h, rstd, x, res, w, eps, cols);
    *launches = 1;
    return (int)cudaGetLastError();
}

extern "C" size_t mcu_rmsnorm_backward_scratch_bytes(int64_t, int64_t) { return 0; }

extern "C" int mcu_launch_rmsnorm_backward(float* dx, float* dw, const float* dy, const float* h, const float* w,
                                           const float* rstd, const float* dh, int64_t rows, int64_t cols, void*,
                                           cudaStream_t st, int* launches) {
    *launches = 0;
    if (dw) {  // first: dx may be dy or h
        rmsnorm_backward_weight<<<(unsigned)((cols + kThreads - 1) / kThreads), kThreads, 0, st>>>(dw, dy, h, rstd, rows, cols);
        ++*launches;
    }
    rmsnorm_backward_row<<<(unsigned)rows, kThreads, 0, st>>>(dx, dy, h, w, rstd, dh, cols);
    ++*launches;
    return (int)cudaGetLastError();
}
