// k_rmsnorm.cu - root-mean-square norm of rows with the residual's addition, f32 and e4m3 outputs, and
// its gradient (mag_cuda_rmsnorm_rows_f32, mag_cuda_rmsnorm_rows_backward_f32).
#include <cuda_runtime.h>
#include <cstdint>
#include "mcu_kernels.h"
#include "mcu_launch.cuh"
#include "mcu_lm.cuh"
#include "mcu_tc.cuh"

using namespace mcu;

namespace {

// Every kernel here gives a warp whole groups of 128 columns (warp w of W: groups w, w + W, ...), so a
// group's largest magnitude is one warp reduction.  A lane holds four of a group's columns: neighbours
// with one 16-byte access (VEC), or columns 32 apart with four 4-byte ones where a row does not start on
// a 16-byte boundary.
template <bool VEC>
__device__ __forceinline__ int lane_col(int lane, int j) { return VEC ? lane * 4 + j : lane + 32 * j; }

// Columns past the row's end read as zero.  (Plain loads: a result may lie over an input.)
template <bool VEC>
__device__ __forceinline__ void load_group(float (&v)[4], const float* p, int c0, int cols, int lane) {
    if (VEC) {
        const float4 t = c0 + lane * 4 < cols ? __ldcs((const float4*)(p + c0 + lane * 4)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        v[0] = t.x;
        v[1] = t.y;
        v[2] = t.z;
        v[3] = t.w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = c0 + lane + 32 * j < cols ? __ldcs(p + c0 + lane + 32 * j) : 0.0f;
    }
}
// The same for values that every row reads again (weights): kept in the caches.
template <bool VEC>
__device__ __forceinline__ void load_weight(float (&v)[4], const float* __restrict__ p, int c0, int cols, int lane) {
    if (VEC) {
        const float4 t = c0 + lane * 4 < cols ? __ldg((const float4*)(p + c0 + lane * 4)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        v[0] = t.x;
        v[1] = t.y;
        v[2] = t.z;
        v[3] = t.w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = c0 + lane + 32 * j < cols ? __ldg(p + c0 + lane + 32 * j) : 0.0f;
    }
}
template <bool VEC>
__device__ __forceinline__ void store_group(float* p, const float (&v)[4], int c0, int cols, int lane) {
    if (VEC) {
        if (c0 + lane * 4 < cols) *(float4*)(p + c0 + lane * 4) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c0 + lane + 32 * j < cols) p[c0 + lane + 32 * j] = v[j];
    }
}

// Sum over the block's warps, the same on every thread.
__device__ __forceinline__ float block_sum(float v, float* sh, int warp, int lane, int warps) {
    v = warp_sum_f(v);
    if (lane == 0) sh[warp] = v;
    __syncthreads();
    return warp_sum_f(lane < warps ? sh[lane] : 0.0f);
}

struct NormArgs {
    float* y;
    uint8_t* q;
    float* s;
    float* h;
    float* rstd;
    const float* x;
    const float* res;
    const float* w;
    float eps;
    int cols;
    int parts;  // blocks of a cluster, which share a row
};
constexpr int kNormCluster = 8;  // at most

// One group's outputs from its sums t.
template <bool VEC>
__device__ __forceinline__ void norm_group(const NormArgs& a, const float (&t)[4], const float (&w)[4], float root,
                                           int64_t row, int g, int groups, int lane) {
    const int64_t o = row * a.cols;
    if (a.h) store_group<VEC>(a.h + o, t, g * 128, a.cols, lane);
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __fmul_rn(__fmul_rn(t[j], root), w[j]);
    if (a.y) store_group<VEC>(a.y + o, v, g * 128, a.cols, lane);
    if (a.q) {
        // past the row's end zero, whatever the root (0 times infinity) and the group (NaN)
        uint32_t keep = 0xFFFFFFFFu;
        if (g * 128 + 128 > a.cols) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (g * 128 + lane_col<VEC>(lane, j) >= a.cols) v[j] = 0.0f, keep &= ~(0xFFu << (8 * j));
        }
        const uint32_t top = __reduce_max_sync(0xffffffffu, max(max(abs_bits(v[0]), abs_bits(v[1])), max(abs_bits(v[2]), abs_bits(v[3]))));
        const E4m3Group gr = e4m3_group(top);
        if (lane == 0) a.s[row * groups + g] = gr.scale;
        const uint32_t b = keep & e4m3_quotients(gr, v[0], v[1], v[2], v[3]);
        uint8_t* q = a.q + (row * groups + g) * 128;
        if (VEC) {
            *(uint32_t*)(q + lane * 4) = b;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) q[lane + 32 * j] = (uint8_t)(b >> (8 * j));
        }
    }
}

// One block of W warps per row, the row held in registers (V groups a warp): one read and one write of
// every value, bound by HBM where rows abound (8192 x 8192 with the residual and an e4m3 result: 154 us,
// 5.7 TB/s, 0.87 of the copy rate) and by latency (loads, one barrier) where they are few.  Rows wider than a
// block's registers are shared by a cluster (CLUSTER), each block a span of the row and one meeting for the sum:
// 4096 x 32768 takes 348 us, 5.0 TB/s (before the e4m3 bytes were decided by two factors 338, and 548 when a second
// pass read the row again), bound by the blocks that an SM holds: four at 64 registers a thread (three at 80 took 6 %
// more).
template <int W, int V, bool VEC, bool CLUSTER = false>
__global__ void __launch_bounds__(W * 32) rmsnorm_row(const NormArgs a) {
    __shared__ float sh[W * (CLUSTER ? kNormCluster : 1)];
    if (CLUSTER) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    pdl_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int parts = CLUSTER ? a.parts : 1, rank = CLUSTER ? (int)blockIdx.x % parts : 0;
    const int64_t row = CLUSTER ? blockIdx.x / (unsigned)parts : blockIdx.x, o = row * a.cols;
    const int groups = (a.cols + 127) >> 7, span = CLUSTER ? (groups + parts - 1) / parts : groups;  // a block's groups
    const int g0 = rank * span + warp, end = CLUSTER ? min(groups, (rank + 1) * span) : groups;
    const int cols = CLUSTER ? min(a.cols, end * 128) : a.cols;
    float t[V][4], w[V][4];
#pragma unroll
    for (int i = 0; i < V; ++i) load_group<VEC>(t[i], a.x + o, (g0 + i * W) * 128, cols, lane);
    if (a.res) {
        float u[V][4];
#pragma unroll
        for (int i = 0; i < V; ++i) load_group<VEC>(u[i], a.res + o, (g0 + i * W) * 128, cols, lane);
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) t[i][j] = __fadd_rn(t[i][j], u[i][j]);
    }
    if (V <= 2) {
#pragma unroll
        for (int i = 0; i < V; ++i) load_weight<VEC>(w[i], a.w, (g0 + i * W) * 128, cols, lane);
    }
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) ss = fmaf(t[i][j], t[i][j], ss);
    float all;
    if (CLUSTER) {  // every warp leaves its share in each block's array
        all = warp_sum_f(ss);
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // every block of the cluster runs
        if (lane < parts)
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(mapa_rank(smem_u32(sh + rank * W + warp), lane)), "f"(all) : "memory");
        __syncwarp();
        cluster_sync();
        all = 0.0f;
        for (int i = lane; i < parts * W; i += 32) all += sh[i];
        all = warp_sum_f(all);
    } else {
        all = block_sum(ss, sh, warp, lane, W);
    }
    const float root = inv_sqrt(__fdiv_rn(all, (float)a.cols) + a.eps);
    if (a.rstd && threadIdx.x == 0 && rank == 0) a.rstd[row] = root;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int g = g0 + i * W;
        if (g >= end) break;
        if (V > 2) load_weight<VEC>(w[i], a.w, g * 128, cols, lane);
        norm_group<VEC>(a, t[i], w[i], root, row, g, groups, lane);
    }
}

// Rows that do not fit a cluster's registers: the second pass reads the row again.
template <bool VEC>
__global__ void __launch_bounds__(1024) rmsnorm_wide(const NormArgs a) {
    __shared__ float sh[32];
    pdl_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row = blockIdx.x, o = row * a.cols;
    const int groups = (a.cols + 127) >> 7;
    const auto sum = [&](float (&t)[4], int g) {
        load_group<VEC>(t, a.x + o, g * 128, a.cols, lane);
        if (a.res) {
            float u[4];
            load_group<VEC>(u, a.res + o, g * 128, a.cols, lane);
#pragma unroll
            for (int j = 0; j < 4; ++j) t[j] = __fadd_rn(t[j], u[j]);
        }
    };
    float ss = 0.0f;
#pragma unroll 4
    for (int g = warp; g < groups; g += 32) {
        float t[4];
        sum(t, g);
#pragma unroll
        for (int j = 0; j < 4; ++j) ss = fmaf(t[j], t[j], ss);
    }
    const float root = inv_sqrt(__fdiv_rn(block_sum(ss, sh, warp, lane, 32), (float)a.cols) + a.eps);
    if (a.rstd && threadIdx.x == 0) a.rstd[row] = root;
    for (int g = warp; g < groups; g += 32) {
        float t[4], w[4];
        sum(t, g);
        load_weight<VEC>(w, a.w, g * 128, a.cols, lane);
        norm_group<VEC>(a, t, w, root, row, g, groups, lane);
    }
}

// ---- the gradient
struct BackArgs {
    float* dx;
    float* part;  // [grid][cols] sums of dy h rstd over a block's rows, or null
    const float* dy;
    const float* h;
    const float* w;
    const float* rstd;
    const float* dh;
    int64_t rows;
    int cols;
    int parts;    // blocks of a cluster, which share every row
    int* status;  // of its bounded waits
    int stall;    // a test of them: nobody sends in the first row
};

constexpr int kBackV = 4;         // groups a warp
constexpr int kBackWarps = 16;    // warps of a block at most
constexpr int kBackAhead = 12;    // and of one that fetches dh a row ahead
constexpr int kBackCluster = 8;   // blocks of a cluster at most

// Sum over the warps of the cluster's blocks, the same on every thread: each warp sends its share to every
// block's sh [parts][kBackWarps], counted on that block's mbarrier.  (A cluster barrier instead would wait for
// the row's stores and loads as well: 4096 x 16384 takes 217 us so, 188 this way.)  Two arrays and mbarriers
// take turns: whoever sends to one again has received what every warp sent after its last reading.  False, for the
// whole warp, when a wait gave up: the warp then leaves the rows, so that no mbarrier is armed again whose phase is
// not complete, and its peers, which get nothing more from it, run out of theirs and follow.
__device__ __forceinline__ bool cluster_sum(float v, float* all, float* sh, uint64_t* bar, uint32_t parity, int warp, int lane, int warps,
                                            int rank, int parts, const Abort& ab, bool send) {
    v = warp_sum_f(v);
    if (threadIdx.x == 0) mbar_expect_tx(bar, (uint32_t)(parts * warps * 4));
    if (lane < parts && send)
        asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.f32 [%0], %1, [%2];" ::"r"(
                         mapa_rank(smem_u32(sh + rank * kBackWarps + warp), lane)),
                     "f"(v), "r"(mapa_rank(smem_u32(bar), lane))
                     : "memory");
    // one lane polls: 32 that give up take 32 times as long, half a second each
    uint32_t ok = 1;
    if (lane == 0) ok = mbar_wait(bar, parity, ab, 24);
    __syncwarp();
    if (!__shfl_sync(0xffffffffu, ok, 0)) return false;
    float t = 0.0f;
    for (int i = lane; i < parts * kBackWarps; i += 32)
        if (i % kBackWarps < warps) t += sh[i];
    *all = warp_sum_f(t);
    return true;
}

// A block goes through rows blockIdx.x, + grid, ...; a thread keeps the same columns in every row and so its
// sums for the weight's gradient in registers.  The next row's dy and h are in flight during the row's
// reduction, which has one barrier: with h loaded after the row's stores instead, every row waited for it
// (4099 x 5000 took 71 us, then 64).  Bound by HBM, 12 bytes read and 4 written a value: 8192 x 8192 runs at
// 6.5 TB/s.  Rows that leave an SM with 9 to 12 warps keep too few bytes in flight that way; their blocks
// have the registers to fetch dh a row ahead too (AHEAD: 58 us, 5.6 TB/s; two blocks an SM with half the
// registers each spilled and took 66 us).  Rows that do not fit a block's registers (8192 columns) are shared
// by a cluster (CLUSTER): 4096 x 12288 in 126 us, 6.4 TB/s; in two passes over the row and one for the weight's
// gradient it took 281.
template <bool VEC, bool AHEAD, bool CLUSTER>
__global__ void __launch_bounds__(32 * (AHEAD ? kBackAhead : kBackWarps), 1) rmsnorm_backward_row(const BackArgs a) {
    constexpr int V = kBackV;
    __shared__ float sh[2][kBackWarps * (CLUSTER ? kBackCluster : 1)];
    __shared__ uint64_t bars[2];
    __shared__ volatile int gave_up;
    const Abort ab{&gave_up, a.status};
    if (CLUSTER) {
        if (threadIdx.x == 0) {
            gave_up = 0;
            mbar_init(&bars[0], 1);
            mbar_init(&bars[1], 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    }
    pdl_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const int parts = CLUSTER ? a.parts : 1, rank = CLUSTER ? (int)blockIdx.x % parts : 0;
    const int first = CLUSTER ? (int)blockIdx.x / parts : (int)blockIdx.x, step = CLUSTER ? (int)gridDim.x / parts : (int)gridDim.x;
    const auto base = [&](int i) { return ((rank * V + i) * warps + warp) * 128; };
    float sum[V][4], dy[V][4], h[V][4];
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[i][j] = 0.0f;
    uint32_t turn = 0;
    int64_t row = first;
    float root = __ldg(a.rstd + row);
#pragma unroll
    for (int i = 0; i < V; ++i) load_group<VEC>(dy[i], a.dy + row * a.cols, base(i), a.cols, lane);
#pragma unroll
    for (int i = 0; i < V; ++i) load_group<VEC>(h[i], a.h + row * a.cols, base(i), a.cols, lane);
    float dh[AHEAD ? V : 1][4];
    if (AHEAD && a.dh) {
#pragma unroll
        for (int i = 0; i < V; ++i) load_group<VEC>(dh[AHEAD ? i : 0], a.dh + row * a.cols, base(i), a.cols, lane);
    }
    if (CLUSTER) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // every block of the cluster runs
    for (; row < a.rows; row += step, ++turn) {
        const int64_t o = row * a.cols, next = row + step;
        float g[V][4], u[V][4], hn[V][4], gn[AHEAD ? V : 1][4];  // the residual path's gradient, then the result; dy w; the next h
        if (!AHEAD && a.dh) {
#pragma unroll
            for (int i = 0; i < V; ++i) load_group<VEC>(g[i], a.dh + o, base(i), a.cols, lane);
        }
        float along = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float w[4];
            load_weight<VEC>(w, a.w, base(i), a.cols, lane);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                u[i][j] = dy[i][j] * w[j];
                along = fmaf(u[i][j], h[i][j], along);
                sum[i][j] = fmaf(dy[i][j], h[i][j] * root, sum[i][j]);
            }
        }
        float next_root = 0.0f;
        if (next < a.rows) {
#pragma unroll
            for (int i = 0; i < V; ++i) load_group<VEC>(dy[i], a.dy + next * a.cols, base(i), a.cols, lane);
#pragma unroll
            for (int i = 0; i < V; ++i) load_group<VEC>(hn[i], a.h + next * a.cols, base(i), a.cols, lane);
            next_root = __ldg(a.rstd + next);
            if (AHEAD && a.dh) {
#pragma unroll
                for (int i = 0; i < V; ++i) load_group<VEC>(gn[AHEAD ? i : 0], a.dh + next * a.cols, base(i), a.cols, lane);
            }
        }
        float all;
        if (CLUSTER) {
            if (!cluster_sum(along, &all, sh[turn & 1], &bars[turn & 1], turn >> 1 & 1, warp, lane, warps, rank, parts, ab, !a.stall || turn))
                break;
        } else {
            all = block_sum(along, sh[turn & 1], warp, lane, warps);
        }
        const float f = root * root * __fdiv_rn(all, (float)a.cols);
#pragma unroll
        for (int i = 0; i < V; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float d = root * fmaf(-h[i][j], f, u[i][j]);
                g[i][j] = a.dh ? __fadd_rn(AHEAD ? dh[AHEAD ? i : 0][j] : g[i][j], d) : d;
                if (AHEAD) dh[AHEAD ? i : 0][j] = gn[AHEAD ? i : 0][j];
                h[i][j] = hn[i][j];
            }
            store_group<VEC>(a.dx + o, g[i], base(i), a.cols, lane);
        }
        root = next_root;
    }
    if (a.part) {
#pragma unroll
        for (int i = 0; i < V; ++i) store_group<VEC>(a.part + (int64_t)first * a.cols, sum[i], base(i), a.cols, lane);
    }
    if (CLUSTER) {
        cluster_sync();  // no block leaves while a peer may still send to it
        if (threadIdx.x == 0 && gave_up)  // and none that did not wait for what was sent before it has had time to land
            for (int i = 0; i < 1024; ++i) __nanosleep(64);
    }
}

// Rows that do not fit a cluster either: dx in two passes over the row, dw's partial sums by columns over a share of rows.
template <bool VEC>
__global__ void __launch_bounds__(1024) rmsnorm_backward_wide(const BackArgs a) {
    __shared__ float sh[32];
    pdl_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row = blockIdx.x, o = row * a.cols;
    const int groups = (a.cols + 127) >> 7;
    const float root = __ldg(a.rstd + row);
    float along = 0.0f;
#pragma unroll 2
    for (int g = warp; g < groups; g += 32) {
        float dy[4], h[4], w[4];
        load_group<VEC>(dy, a.dy + o, g * 128, a.cols, lane);
        load_group<VEC>(h, a.h + o, g * 128, a.cols, lane);
        load_weight<VEC>(w, a.w, g * 128, a.cols, lane);
#pragma unroll
        for (int j = 0; j < 4; ++j) along = fmaf(dy[j] * w[j], h[j], along);
    }
    const float f = root * root * __fdiv_rn(block_sum(along, sh, warp, lane, 32), (float)a.cols);
#pragma unroll 2
    for (int g = warp; g < groups; g += 32) {
        float dy[4], h[4], w[4], t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        load_group<VEC>(dy, a.dy + o, g * 128, a.cols, lane);
        load_group<VEC>(h, a.h + o, g * 128, a.cols, lane);
        load_weight<VEC>(w, a.w, g * 128, a.cols, lane);
        if (a.dh) load_group<VEC>(t, a.dh + o, g * 128, a.cols, lane);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float d = root * fmaf(-h[j], f, dy[j] * w[j]);
            t[j] = a.dh ? __fadd_rn(t[j], d) : d;
        }
        store_group<VEC>(a.dx + o, t, g * 128, a.cols, lane);
    }
}

__global__ void __launch_bounds__(256) rmsnorm_weight_part(const BackArgs a, int64_t col_blocks, int64_t per) {
    pdl_begin();
    const int64_t c = (int64_t)(blockIdx.x % col_blocks) * 256 + threadIdx.x, slice = blockIdx.x / col_blocks;
    if (c >= a.cols) return;
    float t = 0.0f;
    for (int64_t r = slice * per; r < min(slice * per + per, a.rows); ++r)
        t = fmaf(a.dy[r * a.cols + c], a.h[r * a.cols + c] * __ldg(a.rstd + r), t);
    a.part[slice * a.cols + c] = t;
}

// dw = the sum of the partial sums in a fixed order: 32 columns a block, a warp per share of the parts, then
// a warp per column over the shares.
__global__ void __launch_bounds__(1024) rmsnorm_weight_sum(float* __restrict__ dw, const float* __restrict__ part, int parts, int cols) {
    __shared__ float sh[32][33];
    pdl_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = blockIdx.x * 32 + lane, per = (parts + 31) / 32;
    float t = 0.0f;
    if (c < cols) {
#pragma unroll 8
        for (int p = warp * per; p < min(warp * per + per, parts); ++p) t += part[(int64_t)p * cols + c];
    }
    sh[warp][lane] = t;
    __syncthreads();
    t = warp_sum_f(sh[lane][warp]);
    if (lane == 0 && blockIdx.x * 32 + warp < cols) dw[blockIdx.x * 32 + warp] = t;
}

constexpr int kSms = 148;
constexpr int kWideParts = 64;

// Blocks that share a row in the backward pass: rows wider than a block's registers take an even number, since
// clusters of three found no room when the kernel before left the SMs in an odd order (4096 x 16384: 253 us, 187
// in twos).  Blocks of up to 12 warps, which fetch dh ahead, are the faster ones (4096 x 32768: 356 us in sixes,
// 400 in fours), but not by enough to take four instead of two (194 us and 187).
int back_parts(int64_t cols) {
    if (cols <= kBackWarps * kBackV * 128) return 1;
    int parts = 2;
    while (parts < kBackCluster && cols > (int64_t)parts * (parts == 2 ? kBackWarps : kBackAhead) * kBackV * 128) parts += 2;
    return parts;
}
// Warps of a block (0: rows too wide for a cluster's registers), and the rows in work at once: as many as the
// GPU holds (16 warps an SM by their registers).
int back_warps(int64_t cols) {
    const int64_t each = 128 * kBackV * back_parts(cols), w = (cols + each - 1) / each;
    return w <= kBackWarps ? (int)w : 0;
}
int64_t back_blocks(int64_t rows, int64_t cols) {
    if (back_parts(cols) > 1) return rows < kSms / back_parts(cols) ? rows : kSms / back_parts(cols);
    // (few rows: about four a block, or one where that leaves SMs idle, since every block adds a part to dw)
    const int64_t all = kSms * (16 / back_warps(cols)), four = rows < kSms ? rows : rows / 4 > kSms ? rows / 4 : kSms;
    return four < all ? four : all;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// A launch of clusters of `parts` blocks, as a programmatic dependent of the stream's previous kernel.
struct ClusterLaunch {
    cudaLaunchAttribute attr[2] = {};
    cudaLaunchConfig_t cfg = {};
    ClusterLaunch(dim3 grid, dim3 block, int parts, cudaStream_t st) {
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)parts;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.gridDim = grid;
        cfg.blockDim = block;
        cfg.stream = st;
        cfg.attrs = attr;
        cfg.numAttrs = 2;
    }
};

template <typename K>
int go(K kern, int64_t grid, int threads, cudaStream_t st, const NormArgs& a) {
    return (int)launch_dep(kern, dim3((unsigned)grid), dim3((unsigned)threads), 0, st, a);
}
template <bool VEC>
int run_norm(NormArgs& a, int64_t rows, cudaStream_t st) {
    const int groups = (a.cols + 127) / 128;
    // wide rows: a cluster, except where 32 warps of one block are the quicker (300 x 16000: 12.6 us, 14.1 by two
    // blocks; 4096 x 12288: 124 us, 135 by two)
    if (groups <= 64 * kNormCluster && (groups > 128 || (groups > 96 && rows > 4 * kSms))) {
        a.parts = (groups + 63) / 64;
        ClusterLaunch l(dim3((unsigned)(rows * a.parts)), dim3(256), a.parts, st);
        return (int)cudaLaunchKernelEx(&l.cfg, rmsnorm_row<8, 8, VEC, true>, (const NormArgs)a);
    }
    // few rows: 32 warps share a row and each holds less of it
    if (groups > 64 || (rows <= 2 * kSms && groups > 8)) {
        if (groups <= 32) return go(rmsnorm_row<32, 1, VEC>, rows, 1024, st, a);
        if (groups <= 64) return go(rmsnorm_row<32, 2, VEC>, rows, 1024, st, a);
        if (groups <= 128) return go(rmsnorm_row<32, 4, VEC>, rows, 1024, st, a);
        return go(rmsnorm_wide<VEC>, rows, 1024, st, a);
    }
    if (groups <= 8) return go(rmsnorm_row<8, 1, VEC>, rows, 256, st, a);
    if (groups <= 16) return go(rmsnorm_row<8, 2, VEC>, rows, 256, st, a);
    if (groups <= 32) return go(rmsnorm_row<8, 4, VEC>, rows, 256, st, a);
    return go(rmsnorm_row<8, 8, VEC>, rows, 256, st, a);
}

// *blocks: the clusters wanted, lowered to those that the GPU holds at once.
int run_back_cluster(void (*kern)(BackArgs), const BackArgs& a, int* blocks, int warps, cudaStream_t st) {
    ClusterLaunch l(dim3((unsigned)(*blocks * a.parts)), dim3(32u * warps), a.parts, st);
    int held = 0;
    l.cfg.numAttrs = 1;  // the query takes the cluster's shape only
    if (cudaOccupancyMaxActiveClusters(&held, kern, &l.cfg) != cudaSuccess || held <= 0) {
        cudaGetLastError();
        held = *blocks;  // no answer: clusters that do not fit wait for those that do
    }
    if (held < *blocks) *blocks = held;
    l.cfg.gridDim = dim3((unsigned)(*blocks * a.parts));
    l.cfg.numAttrs = 2;
    return (int)cudaLaunchKernelEx(&l.cfg, kern, a);
}
template <bool VEC>
int run_back(const BackArgs& a, int* blocks, cudaStream_t st) {
    const int w = back_warps(a.cols);
    if (!w) return (int)launch_dep(rmsnorm_backward_wide<VEC>, dim3((unsigned)a.rows), dim3(1024), 0, st, a);
    if (a.parts > 1) return run_back_cluster(w <= kBackAhead ? rmsnorm_backward_row<VEC, true, true> : rmsnorm_backward_row<VEC, false, true>, a, blocks, w, st);
    return (int)launch_dep(w > 8 && w <= kBackAhead ? rmsnorm_backward_row<VEC, true, false> : rmsnorm_backward_row<VEC, false, false>,
                           dim3((unsigned)*blocks), dim3(32u * w), 0, st, a);
}

}  // namespace

extern "C" int mcu_launch_rmsnorm(float* y, uint8_t* q, float* s, float* h, float* rstd, const float* x,
                                  const float* res, const float* w, float eps, int64_t rows, int64_t cols,
                                  cudaStream_t st, int* launches) {
    NormArgs a{y, q, s, h, rstd, x, res, w, eps, (int)cols, 1};
    *launches = 1;
    if (cols % 4 == 0 && aligned16(x) && aligned16(res) && aligned16(w) && aligned16(y) && aligned16(h)) return run_norm<true>(a, rows, st);
    return run_norm<false>(a, rows, st);
}

extern "C" size_t mcu_rmsnorm_backward_scratch_bytes(int64_t rows, int64_t cols) {
    return (size_t)((back_warps(cols) ? back_blocks(rows, cols) : kWideParts) * cols) * 4;
}

extern "C" int mcu_launch_rmsnorm_backward(float* dx, float* dw, const float* dy, const float* h, const float* w,
                                           const float* rstd, const float* dh, int64_t rows, int64_t cols, void* scratch,
                                           int* status, cudaStream_t st, int* launches) {
    const BackArgs a{dx, dw ? (float*)scratch : nullptr, dy, h, w, rstd, dh, rows, (int)cols, back_parts(cols), status, test_stall()};
    *launches = 0;
    int parts = back_warps(cols) ? (int)back_blocks(rows, cols) : 0, rc = 0;
    if (dw && !parts) {  // before dx, which may lie over dy or h
        const int64_t cb = (cols + 255) / 256, per = (rows + kWideParts - 1) / kWideParts;
        parts = (int)((rows + per - 1) / per);
        rc = (int)launch_dep(rmsnorm_weight_part, dim3((unsigned)(cb * parts)), dim3(256), 0, st, a, cb, per);
        ++*launches;
    }
    if (!rc) {
        rc = cols % 4 == 0 && aligned16(dx) && aligned16(dy) && aligned16(h) && aligned16(w) && aligned16(dh) ? run_back<true>(a, &parts, st)
                                                                                                               : run_back<false>(a, &parts, st);
        ++*launches;
    }
    if (!rc && dw) {
        rc = (int)launch_dep(rmsnorm_weight_sum, dim3((unsigned)((cols + 31) / 32)), dim3(1024), 0, st, dw, (const float*)a.part, parts, (int)cols);
        ++*launches;
    }
    return rc;
}
