// k_quantize_e4m3.cu - f32 matrices to e4m3 operands with a scale per 1 x 128 or 128 x 128 group, as they
// lie or transposed (mag_cuda_quantize_e4m3).
#include <cuda_runtime.h>
#include <cstdint>
#include "mcu_kernels.h"
#include "mcu_launch.cuh"
#include "mcu_lm.cuh"

using namespace mcu;

namespace {

constexpr int kThreads = 256;  // 8 warps of 16 rows

// Masks the first n bytes of a word.  (Bytes past the matrix are zero, also in a group that a NaN makes NaN.)
__device__ __forceinline__ uint32_t first_bytes(int n) { return n >= 4 ? 0xFFFFFFFFu : n <= 0 ? 0u : (1u << (8 * n)) - 1; }

// One block per 128 x 128 tile of x, in registers: a warp holds 16 of the tile's rows, a lane four of its
// columns (VEC: neighbours, one 16-byte load a row; else 32 apart, four 4-byte loads), all loads issued
// before the first use.  Largest magnitudes are taken over a lane's columns or rows in registers and
// joined by warp reductions and one exchange in shared memory.  Transposed, a lane's 16 rows of a column
// are 16 neighbouring bytes of the result: they go through a 16 KB tile (16-byte pieces, exclusive-or
// swizzled against bank conflicts) and leave as whole 128-byte rows.
// Bound by HBM, 4 bytes read and 1 written a value, with two conversions a value beside it: 8192 x 8192 in rows takes
// 63 us (5.3 TB/s, 0.82 of the copy rate), an 8192 x 4096 weight turned, in blocks, 31.4 us (5.3 TB/s, 0.82).
// A group's scale and factors are formed once: by lane i for the warp's row i, by thread n for the tile's column n.
template <bool VEC, bool BLOCK, bool TRANSPOSE>
__global__ void __launch_bounds__(kThreads, 2) quantize_tile(uint8_t* __restrict__ q, float* __restrict__ s,
                                                             const float* __restrict__ x, int rows, int cols, int col_tiles,
                                                             int64_t ld) {
    __shared__ uint32_t sh_top[TRANSPOSE && !BLOCK ? 8 : 1][TRANSPOSE && !BLOCK ? 128 : 8];
    __shared__ float sh_group[3][TRANSPOSE && !BLOCK ? 128 : 1];
    __shared__ __align__(16) uint8_t tile[TRANSPOSE ? 128 * 128 : 16];
    pdl_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int r0 = (int)(blockIdx.x / col_tiles) * 128, c0 = (int)(blockIdx.x % col_tiles) * 128;
    const int r = r0 + warp * 16;
    const auto col = [&](int j) { return VEC ? lane * 4 + j : lane + 32 * j; };  // of the tile
    float v[16][4];
    const float* p = x + (int64_t)r * cols + c0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        if (VEC) {  // cols is a multiple of 4
            const float4 t = r + i < rows && c0 + lane * 4 < cols ? __ldcs((const float4*)(p + (int64_t)i * cols + lane * 4))
                                                                   : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            v[i][0] = t.x;
            v[i][1] = t.y;
            v[i][2] = t.z;
            v[i][3] = t.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                v[i][j] = r + i < rows && c0 + col(j) < cols ? __ldcs(p + (int64_t)i * cols + col(j)) : 0.0f;
        }
    }
    const int64_t groups = ld / 128;
    E4m3Group gr;  // of the block; of row `lane` of the warp's; of the present column
    if constexpr (BLOCK) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) top = max(top, abs_bits(v[i][j]));
        top = __reduce_max_sync(0xffffffffu, top);
        if (lane == 0) sh_top[0][warp] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, sh_top[0][i]);
        gr = e4m3_group(top);
        if (threadIdx.x == 0) s[TRANSPOSE ? c0 / 128 * groups + r0 / 128 : r0 / 128 * groups + c0 / 128] = gr.scale;
    } else if constexpr (TRANSPOSE) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) top = max(top, abs_bits(v[i][j]));
            sh_top[warp][col(j)] = top;
        }
        __syncthreads();
        if (threadIdx.x < 128) {  // a column each
            const int n = threadIdx.x;
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max(top, sh_top[i][n]);
            const E4m3Group g = e4m3_group(top);
            sh_group[0][n] = g.scale;
            sh_group[1][n] = g.low;
            sh_group[2][n] = g.high;
            if (c0 + n < cols) s[(int64_t)(c0 + n) * groups + r0 / 128] = g.scale;
        }
        __syncthreads();
    } else {
        uint32_t mine = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint32_t top = __reduce_max_sync(
                0xffffffffu, max(max(abs_bits(v[i][0]), abs_bits(v[i][1])), max(abs_bits(v[i][2]), abs_bits(v[i][3]))));
            if (lane == i) mine = top;
        }
        gr = e4m3_group(mine);
        if (lane < 16 && r + lane < rows) s[(int64_t)(r + lane) * groups + c0 / 128] = gr.scale;
    }
    if constexpr (!TRANSPOSE) {
        uint32_t keep = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) keep |= c0 + col(j) < cols ? 0xFFu << (8 * j) : 0u;
        const auto put = [&](int i, uint32_t b) {
            b &= keep;
            uint8_t* o = q + (int64_t)(r + i) * ld + c0;
            if (VEC) {
                *(uint32_t*)(o + lane * 4) = b;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) o[col(j)] = (uint8_t)(b >> (8 * j));
            }
        };
        uint32_t open = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (r + i >= rows) break;  // (for the whole warp)
            if constexpr (BLOCK) {
                put(i, e4m3_quotients(gr, v[i][0], v[i][1], v[i][2], v[i][3]));
            } else {
                const E4m3Group g{0.0f, __shfl_sync(0xffffffffu, gr.low, i), __shfl_sync(0xffffffffu, gr.high, i)};
                put(i, e4m3_try(g, v[i][0], v[i][1], v[i][2], v[i][3], &open));
            }
        }
        if (!BLOCK && __any_sync(0xffffffffu, open)) {  // one warp of a hundred
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                if (r + i >= rows) break;
                put(i, e4m3_divide(__shfl_sync(0xffffffffu, gr.scale, i), v[i][0], v[i][1], v[i][2], v[i][3]));
            }
        }
    } else {
        const auto piece = [&](int n, int c) { return n * 128 + ((c ^ ((VEC ? n >> 2 : n) & 7)) << 4); };
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (!BLOCK) gr = E4m3Group{sh_group[0][col(j)], sh_group[1][col(j)], sh_group[2][col(j)]};
            uint4 b;
            b.x = e4m3_quotients(gr, v[0][j], v[1][j], v[2][j], v[3][j]);
            b.y = e4m3_quotients(gr, v[4][j], v[5][j], v[6][j], v[7][j]);
            b.z = e4m3_quotients(gr, v[8][j], v[9][j], v[10][j], v[11][j]);
            b.w = e4m3_quotients(gr, v[12][j], v[13][j], v[14][j], v[15][j]);
            if (r + 16 > rows) {
                b.x &= first_bytes(rows - r);
                b.y &= first_bytes(rows - r - 4);
                b.z &= first_bytes(rows - r - 8);
                b.w &= first_bytes(rows - r - 12);
            }
            *(uint4*)(tile + piece(col(j), warp)) = b;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int n = warp * 16 + i * 4 + (lane >> 3), c = lane & 7;
            if (c0 + n < cols) *(uint4*)(q + (int64_t)(c0 + n) * ld + r0 + c * 16) = *(const uint4*)(tile + piece(n, c));
        }
    }
}

}  // namespace

extern "C" int mcu_launch_quantize_e4m3(uint8_t* q, float* s, const float* x, int64_t rows, int64_t cols, int block,
                                        int transpose, cudaStream_t st, int* launches) {
    const int64_t ct = (cols + 127) / 128, tiles = (rows + 127) / 128 * ct;
    const int64_t ld = ((transpose ? rows : cols) + 127) / 128 * 128;
    if (tiles > 0x7fffffff) return (int)cudaErrorInvalidValue;
    const bool vec = cols % 4 == 0 && ((uintptr_t)x & 15) == 0;
    const auto go = [&](auto kern) {
        return (int)launch_dep(kern, dim3((unsigned)tiles), dim3(kThreads), 0, st, q, s, x, (int)rows, (int)cols, (int)ct, ld);
    };
    *launches = 1;
    if (vec)
        return transpose ? (block ? go(quantize_tile<true, true, true>) : go(quantize_tile<true, false, true>))
                         : (block ? go(quantize_tile<true, true, false>) : go(quantize_tile<true, false, false>));
    return transpose ? (block ? go(quantize_tile<false, true, true>) : go(quantize_tile<false, false, true>))
                     : (block ? go(quantize_tile<false, true, false>) : go(quantize_tile<false, false, false>));
}
