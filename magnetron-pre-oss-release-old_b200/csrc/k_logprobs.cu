// k_logprobs.cu - log probabilities of given tokens with entropy and the best alternatives, and their
// gradient (mag_cuda_token_logprobs_f32, mag_cuda_token_logprobs_backward_f32).
#include <cuda_runtime.h>
#include <cstdint>
#include "mcu_kernels.h"
#include "mcu_lm.cuh"

using namespace mcu;

namespace {

constexpr int kThreads = 256;

// The order of the alternatives as one integer: larger logit first, then lower column; NaN above
// everything, -0 as +0.
__device__ __forceinline__ uint64_t rank_key(float v, uint32_t col) {
    uint32_t b = __float_as_uint(v + 0.0f);
    b = v != v ? 0xFFFFFFFFu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return (uint64_t)b << 32 | (0xFFFFFFFFu - col);
}

template <typename T, typename F>
__device__ T block_join(T v, F f) {
    __shared__ T sh[kThreads / 32];
    for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh[0];
    for (int i = 1; i < kThreads / 32; ++i) v = f(v, sh[i]);
    return v;
}

// One block per row.
__global__ void __launch_bounds__(kThreads) logprobs_row(float* logp, float* lse, float* entropy, float* top_logp,
                                                         int32_t* top_id, const float* x, const int32_t* id,
                                                         int64_t cols, int64_t x_s1, int top) {
    const int64_t row = blockIdx.x;
    const float* p = x + row * x_s1;
    float m = -INFINITY;
    for (int64_t c = threadIdx.x; c < cols; c += kThreads) m = fmaxf(m, p[c]);
    m = block_join(m, [](float a, float b) { return fmaxf(a, b); });
    float s = 0.0f, t = 0.0f;
    for (int64_t c = threadIdx.x; c < cols; c += kThreads) {
        const float d = p[c] - m, e = expf(d);
        s += e;
        if (!(e == 0.0f)) t += e * d;
    }
    const auto add = [](float a, float b) { return a + b; };
    s = block_join(s, add);
    t = block_join(t, add);
    bool nan = false;
    for (int64_t c = threadIdx.x; c < cols; c += kThreads) nan |= p[c] != p[c];
    nan = __syncthreads_or(nan);
    const bool empty = m == -INFINITY && !nan;  // nothing but -inf
    const float l = empty ? -INFINITY : m + logf(s);
    if (threadIdx.x == 0) {
        if (lse) lse[row] = l;
        if (entropy) entropy[row] = empty ? 0.0f : logf(s) - t / s;
        if (logp) {
            const int32_t i = id[row];
            logp[row] = i < 0 ? 0.0f : i >= cols ? __int_as_float(0x7FC00000) : empty ? -INFINITY : p[i] - l;
        }
    }
    uint64_t last = ~0ull;
    for (int k = 0; k < top; ++k) {
        uint64_t best = 0;
        for (int64_t c = threadIdx.x; c < cols; c += kThreads) {
            const uint64_t key = rank_key(p[c], (uint32_t)c);
            if (key < last && key > best) best = key;
        }
        best = block_join(best, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
        last = best;
        if (threadIdx.x == 0) {
            const uint32_t c = 0xFFFFFFFFu - (uint32_t)best;
            if (top_id) top_id[row * top + k] = (int32_t)c;
            if (top_logp) top_logp[row * top + k] = empty ? -INFINITY : p[c] - l;
        }
    }
}

__global__ void __launch_bounds__(kThreads) logprobs_backward_row(float* dx, const float* x, const int32_t* id,
                                                                  const float* lse, const float* entropy,
                                                                  const float* g_logp, const float* g_entropy,
                                                                  int64_t cols, int64_t x_s1, int64_t dx_s1) {
    const int64_t row = blockIdx.x;
    const float l = lse[row];
    const int32_t i = g_logp ? id[row] : -1;
    const float g = i < 0 ? 0.0f : i >= cols ? __int_as_float(0x7FC00000) : g_logp[row];
    const float ge = g_entropy ? g_entropy[row] : 0.0f, en = g_entropy ? entropy[row] : 0.0f;
    for (int64_t c = threadIdx.x; c < cols; c += kThreads) {
        const float d = x[row * x_s1 + c] - l, p = expf(d);
        float v = l == -INFINITY || p == 0.0f ? 0.0f : -p * (g + ge * (d + en));
        if (c == i && l != -INFINITY) v += g;
        dx[row * dx_s1 + c] = v;
    }
}

}  // namespace

extern "C" int mcu_launch_logprobs(float* logp, float* lse, float* entropy, float* top_logp, int32_t* top_id,
                                   const float* x, const int32_t* id, int64_t rows, int64_t cols, int64_t x_s1, int top,
                                   cudaStream_t st, int* launches) {
    logprobs_row<<<(unsigned)rows, kThreads, 0, st>>>(logp, lse, entropy, top_logp, top_id, x, id, cols, x_s1, top);
    *launches = 1;
    return (int)cudaGetLastError();
}

extern "C" int mcu_launch_logprobs_backward(float* dx, const float* x, const int32_t* id, const float* lse,
                                            const float* entropy, const float* g_logp, const float* g_entropy,
                                            int64_t rows, int64_t cols, int64_t x_s1, int64_t dx_s1, cudaStream_t st,
                                            int* launches) {
    logprobs_backward_row<<<(unsigned)rows, kThreads, 0, st>>>(dx, x, id, lse, entropy, g_logp, g_entropy, cols, x_s1,
                                                               dx_s1);
    *launches = 1;
    return (int)cudaGetLastError();
}
