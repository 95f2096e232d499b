// k_matmul_e4m3.cu - the e4m3 quantiser and the product of e4m3 operands with one scale per 128 of K
// (mag_cuda_quantize_e4m3, mag_cuda_matmul_e4m3).
#include <cuda_runtime.h>
#include <cuda_fp8.h>
#include <cstdint>
#include "mcu_kernels.h"
#include "mcu_lm.cuh"

using namespace mcu;

namespace {

// One block per 128 x 128 tile of the operand (its rows a, its columns b), held in shared memory.
__global__ void __launch_bounds__(256) quantize_tile(uint8_t* q, float* s, const float* x, int64_t a, int64_t b,
                                                     int64_t groups, int block, int transpose) {
    extern __shared__ float tile[];  // [128][129]
    __shared__ uint32_t top;
    const int64_t a0 = (int64_t)(blockIdx.x / groups) * 128, b0 = (int64_t)(blockIdx.x % groups) * 128;
    if (threadIdx.x == 0) top = 0;
    for (int i = threadIdx.x; i < 128 * 128; i += 256) {
        const int u = i >> 7, v = i & 127;  // v runs along x's rows
        const int64_t ia = a0 + (transpose ? v : u), ib = b0 + (transpose ? u : v);
        const float t = ia < a && ib < b ? x[transpose ? ib * a + ia : ia * b + ib] : 0.0f;
        tile[(transpose ? v : u) * 129 + (transpose ? u : v)] = t;
    }
    __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (block) {
        uint32_t m = 0;
        for (int i = threadIdx.x; i < 128 * 128; i += 256) m = max(m, abs_bits(tile[(i >> 7) * 129 + (i & 127)]));
        m = __reduce_max_sync(0xffffffffu, m);
        if (lane == 0) atomicMax(&top, m);
        __syncthreads();
    }
    for (int u = warp; u < 128 && a0 + u < a; u += 8) {
        float v[4];
        uint32_t m = 0;
        for (int i = 0; i < 4; ++i) {
            v[i] = tile[u * 129 + lane * 4 + i];
            m = max(m, abs_bits(v[i]));
        }
        const float sc = e4m3_scale(block ? top : __reduce_max_sync(0xffffffffu, m)), inv = __frcp_rn(sc);
        *(uint32_t*)(q + ((a0 + u) * groups + b0 / 128) * 128 + lane * 4) =
            e4m3x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
        if (lane == 0 && !(block && u)) s[(block ? a0 / 128 : a0 + u) * groups + b0 / 128] = sc;
    }
}

__device__ __forceinline__ float from_e4m3(uint8_t v) {
    __nv_fp8_e4m3 t;
    t.__x = v;
    return (float)t;
}

// 32 x 32 outputs per block of 256, K in steps of 32 through shared memory.
__global__ void __launch_bounds__(256) matmul_e4m3_simple(float* r, const uint8_t* xq, const float* xs,
                                                          const uint8_t* yq, const float* ys, int64_t M, int64_t N,
                                                          int64_t groups, int64_t col_tiles, int y_block) {
    __shared__ float tx[32][33], ty[32][33];
    const int64_t m0 = (int64_t)(blockIdx.x / col_tiles) * 32, n0 = (int64_t)(blockIdx.x % col_tiles) * 32;
    const int c = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t n = n0 + c;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int64_t g = 0; g < groups; ++g) {
        float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int k0 = 0; k0 < 128; k0 += 32) {
            for (int i = 0; i < 4; ++i) {
                const int u = w + 8 * i;
                tx[u][c] = m0 + u < M ? from_e4m3(xq[((m0 + u) * groups + g) * 128 + k0 + c]) : 0.0f;
                ty[u][c] = n0 + u < N ? from_e4m3(yq[((n0 + u) * groups + g) * 128 + k0 + c]) : 0.0f;
            }
            __syncthreads();
            for (int k = 0; k < 32; ++k)
                for (int i = 0; i < 4; ++i) part[i] += tx[w + 8 * i][k] * ty[c][k];
            __syncthreads();
        }
        for (int i = 0; i < 4; ++i) {
            const int64_t m = m0 + w + 8 * i;
            if (m < M && n < N) sum[i] += xs[m * groups + g] * ys[(y_block ? n / 128 : n) * groups + g] * part[i];
        }
    }
    for (int i = 0; i < 4; ++i) {
        const int64_t m = m0 + w + 8 * i;
        if (m < M && n < N) r[m * N + n] = sum[i];
    }
}

}  // namespace

extern "C" int mcu_launch_quantize_e4m3(uint8_t* q, float* s, const float* x, int64_t rows, int64_t cols, int block,
                                        int transpose, cudaStream_t st, int* launches) {
    const int64_t a = transpose ? cols : rows, b = transpose ? rows : cols, groups = (b + 127) / 128;
    const int64_t tiles = (a + 127) / 128 * groups;
    if (tiles > 0x7fffffff) return (int)cudaErrorInvalidValue;
    constexpr int smem = 128 * 129 * 4;
    cudaError_t e = cudaFuncSetAttribute(quantize_tile, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return (int)e;
    quantize_tile<<<(unsigned)tiles, 256, smem, st>>>(q, s, x, a, b, groups, block, transpose);
    *launches = 1;
    return (int)cudaGetLastError();
}

extern "C" size_t mcu_matmul_e4m3_scratch_bytes(int64_t, int64_t, int64_t) { return 0; }

extern "C" int mcu_launch_matmul_e4m3(float* r, const uint8_t* xq, const float* xs, const uint8_t* yq,
                                      const float* ys, int64_t M, int64_t K, int64_t N, int y_block, void*, int*,
                                      cudaStream_t st, int* launches) {
    const int64_t ct = (N + 31) / 32, tiles = (M + 31) / 32 * ct;
    if (tiles > 0x7fffffff) return (int)cudaErrorInvalidValue;
    matmul_e4m3_simple<<<(unsigned)tiles, 256, 0, st>>>(r, xq, xs, yq, ys, M, N, (K + 127) / 128, ct, y_block);
    *launches = 1;
    return (int)cudaGetLastError();
}
