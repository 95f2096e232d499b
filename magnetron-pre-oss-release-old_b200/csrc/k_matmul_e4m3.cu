// k_matmul_e4m3.cu - the product of e4m3 operands with one scale per 128 of K (mag_cuda_matmul_e4m3).
#include <cuda_runtime.h>
#include <cstdint>
#include "mcu_kernels.h"
#include "mcu_tc.cuh"

namespace {

// ------------------------------------------------------------ the product
//
// r = x y^T over groups of 128 of K: S = sum_g xs_g ys_g (xq_g . yq_g).  A group is one 128-byte row of a
// 128-byte-swizzled tile, four tcgen05.mma kind::f8f6f4 of 32 bytes of K each, accumulated from zero in
// one of two TMEM accumulators; the epilogue warps multiply it by the two scales and add it to the sums
// they hold in registers, in f32 with rounding to nearest, while the next group's MMAs run.  (Scales of
// any f32 value cannot ride on the tensor core's own block scaling, which takes powers of two.)

__device__ __forceinline__ void umma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc));
}
__device__ __forceinline__ void umma_f8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc));
}
// D f32, A and B e4m3 (format 0), both K-major.
__host__ __device__ constexpr uint32_t idesc_f8(int m, int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// 16 columns, waited for.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr)
        : "memory");
}
// One lane of a converged warp.  The producer and MMA roles run as whole warps and elect the lane only around
// the issue, so that waits, loop and descriptors stay warp-uniform: with a branch on the lane number around
// the role each MMA took about 80 cycles to issue.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// Whole-warp bounded waits on one or two phases, polled by one lane (a poll by 32 lanes takes twice as
// long), which looks once without blocking first: by then the phase is usually complete.
__device__ __forceinline__ bool mbar_ready(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, const Abort& ab, int code) {
    uint32_t ok = 1;
    if ((threadIdx.x & 31) == 0) ok = mbar_ready(bar, parity) || mbar_wait(bar, parity, ab, code);
    return __shfl_sync(0xffffffffu, ok, 0) != 0;
}
__device__ __forceinline__ bool warp_wait2(uint64_t* bar0, uint32_t parity0, uint64_t* bar1, uint32_t parity1, const Abort& ab, int code) {
    uint32_t ok = 1;
    if ((threadIdx.x & 31) == 0) {
        const bool r0 = mbar_ready(bar0, parity0), r1 = mbar_ready(bar1, parity1);
        if (!r0) ok = mbar_wait(bar0, parity0, ab, code);
        if (!r1 && ok) ok = mbar_wait(bar1, parity1, ab, code + 1);
    }
    return __shfl_sync(0xffffffffu, ok, 0) != 0;
}

// Four f32 of shared memory times s, two packed multiplications (each product rounded to nearest as alone).
__device__ __forceinline__ float4 lds4_times(uint32_t at, float s) {
    float4 v;
    asm volatile(
        "{\n\t.reg .b64 a, b, s;\n\t"
        "ld.shared.v2.b64 {a, b}, [%4];\n\t"
        "mov.b64 s, {%5, %5};\n\t"
        "mul.rn.f32x2 a, a, s;\n\t"
        "mul.rn.f32x2 b, b, s;\n\t"
        "mov.b64 {%0, %1}, a;\n\t"
        "mov.b64 {%2, %3}, b;\n\t}"
        : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
        : "r"(at), "f"(s)
        : "memory");
    return v;
}
__device__ __forceinline__ float lds1(uint32_t a) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}

__device__ __forceinline__ void bar_named(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

// On a give-up: the loads that this thread issued (up to load `it`) have to land before the block ends.
template <int STAGES>
__device__ __forceinline__ void drain_loads(uint64_t* full, uint32_t it) {
    for (uint32_t k = it > STAGES ? it - STAGES : 0; k < it; ++k)
        for (uint32_t i = 0; i < kWaitLimit && !mbar_test(&full[k % STAGES], (k / STAGES) & 1); ++i) __nanosleep(64);
}

// ---- large products: CTA pairs, 256 x 256 tiles, persistent
constexpr int kPairThreads = 512;  // warpgroup 0: producer, MMA issuer, two relays; 1: scales; 2 and 3: epilogue
// 256 * kPairCtrl + 256 * kPairEpi = 512 * kPairLaunch: the epilogue holds 128 sums a thread
constexpr int kPairLaunch = 128, kPairCtrl = 40, kPairEpi = 216;
static_assert(kPairCtrl + kPairEpi == 2 * kPairLaunch, "register split must match the launch");
constexpr int kPanel = 8;      // groups of scales staged at a time
constexpr int kGroupRows = 8;  // 256-row blocks that sweep the columns together, so that operands stay in L2

template <bool YROW>
struct PairCfg {
    static constexpr int STAGES = YROW ? 5 : 6;
    static constexpr int HALF = 128 * 128;  // this CTA's rows of x, or its half of y's, one group
    static constexpr int STAGE = 2 * HALF;
    static constexpr int BARS = STAGES * STAGE;
    static constexpr int SLOTS = BARS + 1024;                      // 8 epilogue warps x 32 x 16 f32
    static constexpr int YS = YROW ? 256 : 2;                      // scales of y per group
    static constexpr int PANEL = (128 + YS) * kPanel * 4;          // x's 128 rows, then y's
    static constexpr int PANELS = SLOTS + 8 * 2048;                // two of them
    static constexpr int SMEM = PANELS + 2 * PANEL + 1024;
    static_assert(SMEM <= 227 * 1024, "must fit shared memory");
};

__device__ __forceinline__ void pair_tile(int t, int num_m, int num_n, int& mb, int& nb) {
    const int per = kGroupRows * num_n, g = t / per, first = g * kGroupRows, rows = min(num_m - first, kGroupRows);
    mb = first + (t - g * per) % rows;
    nb = (t - g * per) / rows;
}

// What bounds it: the group-wise epilogue.  A group is 512 cycles of MMA; its 256 fused multiply-adds per
// scheduler with their TMEM loads and the way accumulator -> relay -> warpgroup -> MMA issuer, 2 of them in
// flight, take about 900, at clocks that the 1 kW limit holds near 1.4 GHz: 8192^3 in 0.56 ms (1.95 PFLOP/s)
// for a few calls and 0.63 ms (1.75) back to back; the MMAs and loads alone took 0.40 and 0.46 ms.
// Measured and not kept: four accumulators of 128 columns (MMAs of N = 128 reach 0.84 of the rate), 16
// epilogue warps of 64 columns (more instructions, 0.67 ms), packed f32x2 multiply-adds (half the
// instructions, the same pipe cycles, more register copies: 0.64 ms and up).
//
// The epilogue waits at a named barrier, never on an mbarrier: a polling loop among its 128 live sums made the
// compiler copy half of them every group.  A relay warp per epilogue warpgroup polls the accumulator's mbarrier
// (bounded) and joins the barrier; four more warps stage the scales, a panel of groups ahead.
template <bool YROW>
__global__ void __maxnreg__(kPairLaunch)
    gemm_e4m3_pair(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_y,
                   const float* __restrict__ xs, const float* __restrict__ ys, float* __restrict__ r, int M, int N, int G,
                   int* status, int stall) {
    using C = PairCfg<YROW>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint64_t* full = (uint64_t*)(smem + C::BARS);
    uint64_t* empty = full + C::STAGES;
    uint64_t* acc_full = empty + C::STAGES;
    uint64_t* acc_empty = acc_full + 2;
    uint64_t* sc_full = acc_empty + 2;
    uint64_t* sc_empty = sc_full + 2;
    uint64_t* drain = sc_empty + 2;
    uint32_t* tmem_slot = (uint32_t*)(drain + 1);
    volatile int* gave_up = (volatile int*)(tmem_slot + 1);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const int num_m = (M + 255) >> 8, num_n = (N + 255) >> 8, tiles = num_m * num_n;
    const Abort ab{gave_up, status};
    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&acc_full[a], 1);
            mbar_init(&acc_empty[a], 16);  // one arrival per epilogue warp of both CTAs
            mbar_init(&sc_full[a], 128);
            mbar_init(&sc_empty[a], 2);  // both relays
        }
        mbar_init(drain, 1);
        *gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    pdl_begin();
    const uint32_t tmem = *tmem_slot;

    if (warp < 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPairCtrl));
        if (warp == 0) {  // ---- TMA producer
            uint32_t it = 0, s = 0, phase = 1;
            // stall, a test of the bounded waits: one for a phase that nothing completes, ahead of every load
            bool ok = !stall || warp_wait(&empty[0], 0, ab, 11);
            for (int t = pair; ok && t < tiles; t += pairs) {
                int mb, nb;
                pair_tile(t, num_m, num_n, mb, nb);
                const int xr = mb * 256 + (int)rank * 128, yr = nb * 256 + (int)rank * 128;
                for (int g = 0; g < G; ++g, ++it) {
                    if (!(ok = warp_wait(&empty[s], phase, ab, 11))) break;
                    if (elect_one()) {
                        // both CTAs' loads complete on the leader's barrier, which expects both
                        const uint32_t fb = mapa_rank(smem_u32(&full[s]), 0);
                        uint8_t* st = smem + s * C::STAGE;
                        if (rank == 0) mbar_expect_tx(&full[s], 2 * C::STAGE);
                        tma_load_2d_pair(&map_x, fb, st, g * 128, xr);
                        tma_load_2d_pair(&map_y, fb, st + C::HALF, g * 128, yr);
                    }
                    __syncwarp();
                    if (++s == C::STAGES) s = 0, phase ^= 1;
                }
            }
            if (!ok && rank == 0 && lane == 0) drain_loads<C::STAGES>(full, it);
        } else if (warp == 1) {
            if (rank == 0) {  // ---- MMA issuer, for both CTAs
                constexpr uint32_t idesc = idesc_f8(256, 256);
                const uint64_t first = sw_desc<128>(smem_u32(smem));
                uint32_t it = 0, s = 0, phase = 0;
                bool ok = true;
                for (int t = pair; ok && t < tiles; t += pairs) {
                    for (int g = 0; g < G; ++g, ++it) {
                        const uint32_t b = it & 1;
                        if (!(ok = warp_wait2(&acc_empty[b], (it >> 1 & 1) ^ 1, &full[s], phase, ab, 12))) break;
                        tc_fence_after();
                        const uint64_t dx = first + s * (C::STAGE >> 4), dy = dx + (C::HALF >> 4);
                        if (elect_one()) {
#pragma unroll
                            for (int k = 0; k < 4; ++k) umma_f8_pair(tmem + b * 256, dx + k * 2, dy + k * 2, idesc, k);
                            umma_commit_pair(&acc_full[b]);
                            umma_commit_pair(&empty[s]);
                        }
                        __syncwarp();
                        if (++s == C::STAGES) s = 0, phase ^= 1;
                    }
                }
            }
        } else if (warp < 4) {  // ---- relay of epilogue warpgroup `half`
            const int half = warp - 2;
            uint32_t it = 0, pi = 0;
            for (int t = pair; t < tiles; t += pairs) {
                for (int g = 0; g < G; ++g, ++it) {
                    const bool first = (g & (kPanel - 1)) == 0;
                    // (a relay that gives up goes on without waiting, so that the named barriers stay matched)
                    if (first) warp_wait(&sc_full[pi & 1], pi >> 1 & 1, ab, 20);
                    warp_wait(&acc_full[it & 1], it >> 1 & 1, ab, 14);
                    tc_fence_after();
                    tc_fence_before();
                    bar_named(1 + half, 160);
                    if (first) {  // the warpgroup is past the panel before this one
                        if (pi && lane == 0) mbar_arrive(&sc_empty[(pi & 1) ^ 1]);
                        ++pi;
                    }
                }
            }
        } else {  // ---- scales: thread i brings x's row i of the CTA and y's columns i and i + 128
            const int i = threadIdx.x - 128;
            uint32_t pi = 0;
            bool ok = true;
            for (int t = pair; ok && t < tiles; t += pairs) {
                int mb, nb;
                pair_tile(t, num_m, num_n, mb, nb);
                const float* px = xs + (int64_t)min(mb * 256 + (int)rank * 128 + i, M - 1) * G;
                const float* py0 = ys + (int64_t)(YROW ? min(nb * 256 + i, N - 1) : min(nb * 256 + (i & 1) * 128, N - 1) >> 7) * G;
                const float* py1 = ys + (int64_t)min(nb * 256 + 128 + i, N - 1) * G;  // (scales per row only)
                for (int g0 = 0; g0 < G; g0 += kPanel, ++pi) {
                    const int n = min(kPanel, G - g0);
                    float v[kPanel];
#pragma unroll
                    for (int k = 0; k < kPanel; ++k) v[k] = k < n ? __ldg(px + g0 + k) : 0.0f;
                    if (!(ok = warp_wait(&sc_empty[pi & 1], (pi >> 1 & 1) ^ 1, ab, 19))) break;
                    float* p = (float*)(smem + C::PANELS + (pi & 1) * C::PANEL);
#pragma unroll
                    for (int k = 0; k < kPanel; ++k) p[k * 128 + i] = v[k];
                    p += 128 * kPanel;
                    if constexpr (YROW) {
#pragma unroll
                        for (int k = 0; k < kPanel; ++k) v[k] = k < n ? __ldg(py0 + g0 + k) : 0.0f;
#pragma unroll
                        for (int k = 0; k < kPanel; ++k) p[k * 256 + i] = v[k];
#pragma unroll
                        for (int k = 0; k < kPanel; ++k) v[k] = k < n ? __ldg(py1 + g0 + k) : 0.0f;
#pragma unroll
                        for (int k = 0; k < kPanel; ++k) p[k * 256 + 128 + i] = v[k];
                    } else if (i < 2 * n) {
                        p[i] = __ldg(py0 + g0 + (i >> 1));
                    }
                    mbar_arrive(&sc_full[pi & 1]);
                }
            }
        }
    } else {  // ---- epilogue: lane = row, warpgroup = half of the columns
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPairEpi));
        const int q = warp & 3, half = (warp >> 2) - 2;
        const uint32_t src0 = tmem + ((uint32_t)(q * 32) << 16) + half * 128;
        const uint32_t slot = smem_u32(smem + C::SLOTS + (warp - 8) * 2048);
        const uint32_t panels = smem_u32(smem + C::PANELS);
        const uint32_t released = mapa_rank(smem_u32(&acc_empty[0]), 0);
        const bool vec = (N & 3) == 0 && ((uintptr_t)r & 15) == 0;
        uint32_t it = 0, pi = 0;
        for (int t = pair; t < tiles; t += pairs) {
            int mb, nb;
            pair_tile(t, num_m, num_n, mb, nb);
            const int row0 = mb * 256 + (int)rank * 128 + q * 32, col0 = nb * 256 + half * 128;
            float sum[128];
#pragma unroll
            for (int j = 0; j < 128; ++j) sum[j] = 0.0f;
            for (int g = 0; g < G; ++g, ++it) {
                const uint32_t panel = panels + ((pi + (g / kPanel)) & 1) * C::PANEL + (g & (kPanel - 1)) * 512;
                const uint32_t src = src0 + (it & 1) * 256;
                bar_named(1 + half, 160);
                tc_fence_after();
                float sc = lds1(panel + (q * 32 + lane) * 4);
                const uint32_t py = panels + ((pi + (g / kPanel)) & 1) * C::PANEL + kPanel * 512 + (g & (kPanel - 1)) * C::YS * 4;
                if (!YROW) sc = __fmul_rn(sc, lds1(py + half * 4));
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t v[32];
                    tmem_ld32(src + c * 32, v);
                    if (c == 3) {  // everything is read: the accumulator goes back to the leader's MMA issuer
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_cluster(released + (it & 1) * 8);
                    }
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        float4 s = make_float4(sc, sc, sc, sc);
                        if (YROW) s = lds4_times(py + (half * 128 + c * 32 + j) * 4, sc);
                        float* d = sum + c * 32 + j;
                        d[0] = __fmaf_rn(__uint_as_float(v[j]), s.x, d[0]);
                        d[1] = __fmaf_rn(__uint_as_float(v[j + 1]), s.y, d[1]);
                        d[2] = __fmaf_rn(__uint_as_float(v[j + 2]), s.z, d[2]);
                        d[3] = __fmaf_rn(__uint_as_float(v[j + 3]), s.w, d[3]);
                    }
                }
            }
            pi += (G + kPanel - 1) / kPanel;
            // 32 x 16 chunks through this warp's slot, so that rows leave in pieces of 64 bytes
            const bool ok = !*gave_up;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const int col = col0 + c * 16;
                if (!ok || row0 >= M || col >= N) break;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    sts4(slot + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4), sum[c * 16 + j * 4], sum[c * 16 + j * 4 + 1],
                         sum[c * 16 + j * 4 + 2], sum[c * 16 + j * 4 + 3]);
                __syncwarp();
                if (vec) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int rr = 8 * i + (lane >> 2), cc = lane & 3;
                        const float4 o = lds4(slot + rr * 64 + ((cc ^ ((rr >> 1) & 3)) << 4));
                        if (row0 + rr < M && col + cc * 4 < N) __stcs((float4*)(r + (int64_t)(row0 + rr) * N + col + cc * 4), o);
                    }
                } else {
#pragma unroll 1
                    for (int i = 0; i < 16; ++i) {
                        const int rr = 2 * i + (lane >> 4), cc = lane & 15;
                        const float o = lds1(slot + rr * 64 + (((cc >> 2) ^ ((rr >> 1) & 3)) << 4) + (cc & 3) * 4);
                        if (row0 + rr < M && col + cc < N) r[(int64_t)(row0 + rr) * N + col + cc] = o;
                    }
                }
                __syncwarp();
            }
        }
    }
    __syncthreads();
    if (warp == 1 && rank == 0 && *gave_up && elect_one()) {  // MMAs in flight end before the accumulators go
        umma_commit_pair_local(drain);
        for (uint32_t i = 0; i < kWaitLimit && !mbar_test(drain, 0); ++i) __nanosleep(64);
    }
    __syncwarp();
    tc_fence_before();
    cluster_sync();  // neither CTA leaves while its peer may still signal it or write its TMEM
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
    }
}

// ---- few rows of x: one CTA per 128 rows of y (the MMA's rows) and BN rows of x, K split over a cluster
constexpr int kNarrowAcc = 4;     // accumulators, so that the MMAs run ahead of the epilogue
constexpr int kNarrowPanel = 16;  // groups of x's scales staged at a time

template <int BN, bool YROW>
struct NarrowCfg {
    static constexpr int A = 128 * 128, B = BN * 128, STAGE = A + B;
    static constexpr int STAGES = BN == 32 ? 5 : 6;
    static constexpr int PER_SM = BN <= 32 ? 2 : 1;
    // epilogue warps: four quadrants of lanes, 16 or 32 columns each (BN = 64, N = 14336: 13.2 us with 16 warps, 13.4
    // with 8; with scales of y per row, which each warp fetches, 16.5 and 14.5)
    static constexpr int EPI = BN >= 128 ? 16 : BN == 64 ? (YROW ? 8 : 16) : 4;
    static constexpr int WC = BN * 4 / EPI;       // columns of a warp
    static constexpr int THREADS = 64 + 32 * EPI;
    // scales of y per row: staged like x's where the epilogue's warps are many; the few warps of a narrow tile
    // fetch their own (4 x 4096 x 4096: 5.7 us, 6.9 staged; 100 x 4096 x 14336: 22.4 us, 18.9 staged)
    static constexpr bool STAGE_Y = YROW && BN >= 128;
    static constexpr int PANEL = STAGES * STAGE;  // kNarrowPanel x BN scales of x, then x 128 of y
    static constexpr int BARS = PANEL + kNarrowPanel * (BN + (STAGE_Y ? 128 : 0)) * 4;
    static constexpr int SMEM = BARS + 512 + 1024;
    static constexpr int COLS = kNarrowAcc * BN;
    static_assert(PER_SM * SMEM <= 227 * 1024 && 128 * BN * 4 <= STAGES * STAGE, "must fit shared memory");
};
template <int BN, bool YROW>
__global__ void __launch_bounds__(NarrowCfg<BN, YROW>::THREADS, NarrowCfg<BN, YROW>::PER_SM)
    gemm_e4m3_narrow(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_y,
                     const float* __restrict__ xs, const float* __restrict__ ys, float* __restrict__ r, int M, int N, int G,
                     int parts, int per, int* status, int stall) {
    using C = NarrowCfg<BN, YROW>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint64_t* full = (uint64_t*)(smem + C::BARS);
    uint64_t* empty = full + C::STAGES;
    uint64_t* acc_full = empty + C::STAGES;
    uint64_t* acc_empty = acc_full + kNarrowAcc;
    uint64_t* drain = acc_empty + kNarrowAcc;
    uint32_t* tmem_slot = (uint32_t*)(drain + 1);
    volatile int* gave_up = (volatile int*)(tmem_slot + 1);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int mt = (M + BN - 1) / BN;
    const int part = blockIdx.x % parts, tile = blockIdx.x / parts;
    const int m0 = tile % mt * BN, n0 = tile / mt * 128;
    const int g0 = min(part * per, G), g1 = min(g0 + per, G), ng = g1 - g0;
    const Abort ab{gave_up, status};
    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int a = 0; a < kNarrowAcc; ++a) {
            mbar_init(&acc_full[a], 1);
            mbar_init(&acc_empty[a], C::EPI);
        }
        mbar_init(drain, 1);
        *gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)C::COLS));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_begin();
    const uint32_t tmem = *tmem_slot;
    bool ok = true;

    if (warp == 0) {  // ---- TMA producer
        uint32_t s = 0, phase = 1;
        if (stall) ok = warp_wait(&empty[0], 0, ab, 15);  // (as in the pairs)
        for (int g = g0; ok && g < g1; ++g) {
            if (!(ok = warp_wait(&empty[s], phase, ab, 15))) break;
            if (elect_one()) {
                mbar_expect_tx(&full[s], C::STAGE);
                tma_load_2d(&map_y, &full[s], smem + s * C::STAGE, g * 128, n0);
                tma_load_2d(&map_x, &full[s], smem + s * C::STAGE + C::A, g * 128, m0);
            }
            __syncwarp();
            if (++s == C::STAGES) s = 0, phase ^= 1;
        }
        // (a producer that gives up has at most the ring's loads in flight: they land before the block ends)
        if (!ok && lane == 0)
            for (int k = 0; k < C::STAGES; ++k)
                for (uint32_t i = 0; i < kWaitLimit && !mbar_test(&full[k], k < (int)s ? phase ^ 1 : phase); ++i) __nanosleep(64);
    } else if (warp == 1) {  // ---- MMA issuer
        constexpr uint32_t idesc = idesc_f8(128, BN);
        const uint64_t first = sw_desc<128>(smem_u32(smem));
        uint32_t s = 0, phase = 0;
        for (uint32_t it = 0; it < (uint32_t)ng; ++it) {
            const uint32_t b = it % kNarrowAcc, ap = it / kNarrowAcc & 1;
            if (!(ok = warp_wait2(&acc_empty[b], ap ^ 1, &full[s], phase, ab, 16))) break;
            tc_fence_after();
            const uint64_t dy = first + s * (C::STAGE >> 4), dx = dy + (C::A >> 4);
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < 4; ++k) umma_f8(tmem + b * BN, dy + k * 2, dx + k * 2, idesc, k);
                umma_commit(&acc_full[b]);
                umma_commit(&empty[s]);
            }
            __syncwarp();
            if (++s == C::STAGES) s = 0, phase ^= 1;
        }
    } else {  // ---- epilogue: lane = row of y, warps 6.. the second half of the columns
        const int q = warp & 3, col = ((warp - 2) >> 2) * C::WC, tid = threadIdx.x - 64;
        const int n = n0 + q * 32 + lane;
        const float* py = ys + (int64_t)(YROW ? min(n, N - 1) : n0 >> 7) * G + g0;
        float* panel = (float*)(smem + C::PANEL);
        float sum[C::WC];  // this lane's row of y against the warp's rows of x
#pragma unroll
        for (int j = 0; j < C::WC; ++j) sum[j] = 0.0f;
        // the scales of x's BN rows (a block's scale of y already multiplied in) and of y's 128 rows, 16 groups
        // at a time, fetched one panel ahead
        constexpr int PX = BN * kNarrowPanel / (32 * C::EPI), PY = C::STAGE_Y ? 128 * kNarrowPanel / (32 * C::EPI) : 0;
        float ahead[PX + PY];
        const auto fetch = [&](int it) {
#pragma unroll
            for (int i = 0; i < PX; ++i) {
                const int e = tid + i * 32 * C::EPI, m = m0 + e / kNarrowPanel, g = it + e % kNarrowPanel;
                const bool in = m < M && g < ng;
                ahead[i] = in ? __ldg(xs + (int64_t)m * G + g0 + g) : 0.0f;
                if (!YROW && in) ahead[i] = __fmul_rn(ahead[i], __ldg(py + g));
            }
#pragma unroll
            for (int i = 0; i < PY; ++i) {
                const int e = tid + i * 32 * C::EPI, y = n0 + e / kNarrowPanel, g = it + e % kNarrowPanel;
                ahead[PX + i] = y < N && g < ng ? __ldg(ys + (int64_t)y * G + g0 + g) : 0.0f;
            }
        };
        fetch(0);
        float own_y = YROW && !C::STAGE_Y && ng > 0 ? __ldg(py) : 1.0f;
        bool ready = false;
        for (uint32_t it = 0; it < (uint32_t)ng; ++it) {
            const uint32_t b = it % kNarrowAcc, ap = it / kNarrowAcc & 1;
            if ((it & (kNarrowPanel - 1)) == 0) {
                if (it) bar_named(1, 32 * C::EPI);
#pragma unroll
                for (int i = 0; i < PX + PY; ++i) {
                    const int e = tid + (i < PX ? i : i - PX) * 32 * C::EPI, row = e / kNarrowPanel, g = e % kNarrowPanel;
                    panel[i < PX ? g * BN + row : kNarrowPanel * BN + g * 128 + row] = ahead[i];
                }
                bar_named(1, 32 * C::EPI);
                if (it + kNarrowPanel < (uint32_t)ng) fetch(it + kNarrowPanel);
            }
            const float ay = C::STAGE_Y ? panel[kNarrowPanel * BN + (it & (kNarrowPanel - 1)) * 128 + q * 32 + lane] : own_y;
            if (YROW && !C::STAGE_Y && it + 1 < (uint32_t)ng) own_y = __ldg(py + it + 1);
            // (a warp that gives up goes on without waiting, so that the named barriers stay matched)
            if (!ready) ok &= warp_wait(&acc_full[b], ap, ab, 18);
            tc_fence_after();
            const uint32_t pan = smem_u32(panel + (it & (kNarrowPanel - 1)) * BN + col);
            const uint32_t src = tmem + ((uint32_t)(q * 32) << 16) + b * BN + col;
            uint32_t v[32];
            if constexpr (C::WC == 16) tmem_ld16(src, v);
            else tmem_ld32(src, v);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[b]);
            // the next accumulator is usually complete: looked at here, ahead of the sums
            ready = it + 1 < (uint32_t)ng && __all_sync(0xffffffffu, mbar_ready(&acc_full[(it + 1) % kNarrowAcc], (it + 1) / kNarrowAcc & 1));
#pragma unroll
            for (int j = 0; j < C::WC; j += 4) {
                const float4 x4 = YROW ? lds4_times(pan + j * 4, ay) : lds4(pan + j * 4);
                const uint32_t* w = v + j;
                sum[j] = __fmaf_rn(__uint_as_float(w[0]), x4.x, sum[j]);
                sum[j + 1] = __fmaf_rn(__uint_as_float(w[1]), x4.y, sum[j + 1]);
                sum[j + 2] = __fmaf_rn(__uint_as_float(w[2]), x4.z, sum[j + 2]);
                sum[j + 3] = __fmaf_rn(__uint_as_float(w[3]), x4.w, sum[j + 3]);
            }
        }
        if (ok && parts == 1 && n < N) {
#pragma unroll
            for (int j = 0; j < C::WC; ++j)
                if (m0 + col + j < M) r[(int64_t)(m0 + col + j) * N + n] = sum[j];
        }
        if (ok && parts > 1) {  // the last accumulator was complete, so no MMA reads the ring: it holds the sums now
            float* own = (float*)smem;
#pragma unroll
            for (int j = 0; j < C::WC; ++j) own[(col + j) * 128 + q * 32 + lane] = sum[j];
        }
    }
    __syncthreads();
    if (parts > 1) {
        __syncwarp();
        cluster_sync();
        const bool good = !*gave_up;
        // columns are shared out over the cluster; the parts are added in their order
        for (int i = part * C::THREADS + threadIdx.x; good && i < 128 * BN; i += C::THREADS * parts) {
            const int m = m0 + (i >> 7), n = n0 + (i & 127);
            if (m >= M || n >= N) continue;
            const uint32_t at = smem_u32(smem) + i * 4;
            float a = 0.0f;
            for (int p = 0; p < parts; ++p) {
                float v;
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_rank(at, p)) : "memory");
                a = __fadd_rn(a, v);
            }
            r[(int64_t)m * N + n] = a;
        }
        __syncwarp();
        cluster_sync();  // a CTA's sums stay until every peer has read them
    }
    if (warp == 1) {
        if (*gave_up && elect_one()) {
            umma_commit(drain);
            for (uint32_t i = 0; i < kWaitLimit && !mbar_test(drain, 0); ++i) __nanosleep(64);
        }
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)C::COLS));
    }
}

// ------------------------------------------------------------ host side
// 2-D map over an operand's bytes [rows][ld], box 128 bytes x box_rows, 128-byte swizzle; rows past the
// end read as zero.
bool e4m3_map(CUtensorMap* m, const uint8_t* q, int64_t rows, int64_t ld, int box_rows) {
    auto fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[2] = {(cuuint64_t)ld, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld};
    cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void*)q, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int sms() {
    static int n = 0;
    if (!n) {
        int dev = 0;
        cudaGetDevice(&dev);
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    }
    return n > 0 ? n : 148;
}

// A launch with a cluster of `cluster` CTAs, as a programmatic dependent of the stream's previous kernel.
template <auto kern, typename... A>
int launch(int64_t grid, int threads, int smem, int cluster, cudaStream_t st, A... args) {
    static bool done[64];
    cudaError_t e = allow_smem(kern, smem, done);
    if (e != cudaSuccess) return (int)e;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return (int)cudaLaunchKernelEx(&cfg, kern, args...);
}

template <bool YROW>
int run_pair(const CUtensorMap& mx, const CUtensorMap& my, const float* xs, const float* ys, float* r, int64_t M, int64_t N,
             int64_t G, int* status, cudaStream_t st) {
    const int64_t tiles = (M + 255) / 256 * ((N + 255) / 256);
    if (tiles > 0x7fffffff) return (int)cudaErrorInvalidValue;
    const int64_t pairs = tiles < sms() / 2 ? tiles : sms() / 2;
    return launch<gemm_e4m3_pair<YROW>>(2 * pairs, kPairThreads, PairCfg<YROW>::SMEM, 2, st, mx, my, xs, ys, r, (int)M, (int)N,
                  (int)G, status, test_stall());
}

// CTAs per tile: up to 8, while they all run at once and have at least four groups each
// (K = 2048, N = 4096, M = 4: 4 CTAs 4.5 us, 8 of two groups 4.95).
template <int BN>
int narrow_parts(int64_t tiles, int64_t G) {
    int parts = 1;
    while (parts < 8 && tiles * parts * 2 <= sms() * NarrowCfg<BN, false>::PER_SM && G >= 8 * parts) parts *= 2;
    return parts;
}

template <int BN>
int run_narrow(const CUtensorMap& mx, const CUtensorMap& my, const float* xs, const float* ys, float* r, int64_t M, int64_t N,
               int64_t G, int y_block, int* status, cudaStream_t st) {
    const int64_t tiles = (M + BN - 1) / BN * ((N + 127) / 128);
    const int parts = narrow_parts<BN>(tiles, G);
    if (tiles * parts > 0x7fffffff) return (int)cudaErrorInvalidValue;
    const int per = (int)((G + parts - 1) / parts);
    if (y_block)
        return launch<gemm_e4m3_narrow<BN, false>>(tiles * parts, NarrowCfg<BN, false>::THREADS, NarrowCfg<BN, false>::SMEM, parts, st, mx, my, xs, ys, r, (int)M,
                      (int)N, (int)G, parts, per, status, test_stall());
    return launch<gemm_e4m3_narrow<BN, true>>(tiles * parts, NarrowCfg<BN, true>::THREADS, NarrowCfg<BN, true>::SMEM, parts, st, mx, my, xs, ys, r, (int)M,
                  (int)N, (int)G, parts, per, status, test_stall());
}

// Both kernels run in waves of the GPU: 148 tiles of 128 x 128 at a time, or 74 of 256 x 256.  Measured with
// N = 4096 and 14336 and K = 256 to 8192: a narrow wave takes 4 us and 0.41 us a group of K (0.47 with
// scales of y per row); the persistent pairs take 8.5 us in all and 0.46 us a group and wave (7.3 and 0.80).
// So the pairs win once their larger tiles fill a wave: 512 x 4096 x 4096 takes 17 us narrow and 23 in
// pairs, 1024 x 4096 x 4096 33 us narrow and 23 in pairs.
bool pair_is_faster(int64_t M, int64_t N, int64_t G, int y_block) {
    const int64_t narrow = (M + 127) / 128 * ((N + 127) / 128), pair = (M + 255) / 256 * ((N + 255) / 256), n = sms();
    const int64_t parts = narrow_parts<128>(narrow, G), per = (G + parts - 1) / parts;
    const int64_t tn = (narrow * parts + n - 1) / n * (400 + (y_block ? 41 : 47) * per);
    const int64_t tp = (pair + n / 2 - 1) / (n / 2) * (y_block ? 46 : 80) * G + (y_block ? 850 : 730);
    return tp < tn;
}

}  // namespace

extern "C" int mcu_launch_matmul_e4m3(float* r, const uint8_t* xq, const float* xs, const uint8_t* yq,
                                      const float* ys, int64_t M, int64_t K, int64_t N, int y_block, int* status,
                                      cudaStream_t st, int* launches) {
    const int64_t G = (K + 127) / 128, ld = G * 128;
    const int bn = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : !pair_is_faster(M, N, G, y_block) ? 128 : 0;
    CUtensorMap mx, my;
    if (!e4m3_map(&mx, xq, M, ld, bn ? bn : 128) || !e4m3_map(&my, yq, N, ld, 128)) return (int)cudaErrorInvalidValue;
    *launches = 1;
    switch (bn) {
        case 16: return run_narrow<16>(mx, my, xs, ys, r, M, N, G, y_block, status, st);
        case 32: return run_narrow<32>(mx, my, xs, ys, r, M, N, G, y_block, status, st);
        case 64: return run_narrow<64>(mx, my, xs, ys, r, M, N, G, y_block, status, st);
        case 128: return run_narrow<128>(mx, my, xs, ys, r, M, N, G, y_block, status, st);
        default:
            return y_block ? run_pair<false>(mx, my, xs, ys, r, M, N, G, status, st)
                           : run_pair<true>(mx, my, xs, ys, r, M, N, G, status, st);
    }
}
