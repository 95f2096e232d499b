// k_logprobs.cu - log probabilities of given tokens with entropy and the best alternatives, and their
// gradient (mag_cuda_token_logprobs_f32, mag_cuda_token_logprobs_backward_f32).
//
// With m a maximum and d = x - m, a part of a row is described by S = sum e^d and T = sum e^d d; parts
// join by bringing both to the larger maximum, S' = S e^c and T' = (T + c S) e^c with c = m - m', so one
// pass over the row serves
//   lse = m + ln S,  logp = x[id] - lse,  entropy = ln S - T / S.
// The same pass keeps the row's best candidates: everything above the k-th best seen so far.
#include <cuda_runtime.h>
#include <cooperative_groups.h>
#include <cfloat>
#include <cstdint>
#include "mcu_kernels.h"
#include "mcu_lm.cuh"

namespace cg = cooperative_groups;
using namespace mcu;

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFar = -1e30f;  // stands for d = -inf where it meets a factor of zero
constexpr int kVecs = 4;        // float4 per thread and chunk
constexpr int kMaxCluster = 8;  // CTAs that share a row

__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// The order of the alternatives as one integer: larger logit first, then lower column; NaN above
// everything, -0 as +0.  0 stands for no element.
__device__ __forceinline__ uint64_t rank_key(float v, uint32_t col) {
    uint32_t b = __float_as_uint(v + 0.0f);
    b = v != v ? 0xFFFFFFFFu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return (uint64_t)b << 32 | (0xFFFFFFFFu - col);
}
__device__ __forceinline__ float key_value(uint64_t key) {
    const uint32_t b = (uint32_t)(key >> 32);
    return __uint_as_float((b & 0x80000000u) ? b & 0x7FFFFFFFu : ~b);
}

// Four logits of a row whose first one lies `off` floats past a 16-byte boundary: vector vi holds the
// elements 4 vi - off .. + 3.  Only the first and the last one reach past the row; their elements there
// are -inf, and nothing outside the row is read.
__device__ __forceinline__ float4 load_logits(const float* p, int64_t vi, int64_t nvec, int off, int64_t cols) {
    const int64_t c = vi * 4 - off;
    if (c >= 0 && c + 4 <= cols) return __ldcs((const float4*)(p + c));
    float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    if (vi >= nvec) return v;
    if (c >= 0 && c < cols) v.x = p[c];
    if (c + 1 >= 0 && c + 1 < cols) v.y = p[c + 1];
    if (c + 2 >= 0 && c + 2 < cols) v.z = p[c + 2];
    if (c + 3 >= 0 && c + 3 < cols) v.w = p[c + 3];
    return v;
}

struct Part {
    float m;
    double s, t;
};
__device__ __forceinline__ Part join(const Part& a, const Part& b) {
    const float m = fmaxf(a.m, b.m);
    // (a part of nothing has s = t = 0 and the lowest maximum; the bounded distance keeps 0 * distance at 0)
    const float ca = fmaxf(a.m - m, kFar), cb = fmaxf(b.m - m, kFar);
    const double ea = (double)expf(ca), eb = (double)expf(cb);
    // a maximum of infinity, or NaN terms, leave s NaN
    return Part{m, a.s * ea + b.s * eb, (a.t + ca * a.s) * ea + (b.t + cb * b.s) * eb};
}

// Best 32 of a warp's 32 keys in descending order over the lanes, and of two such lists.
__device__ __forceinline__ uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint64_t min64(uint64_t a, uint64_t b) { return a < b ? a : b; }
__device__ __forceinline__ uint64_t order_bitonic(uint64_t k, int lane) {
#pragma unroll
    for (int j = 16; j; j >>= 1) {
        const uint64_t o = __shfl_xor_sync(0xffffffffu, k, j);
        k = (lane & j) ? min64(k, o) : max64(k, o);
    }
    return k;
}
__device__ __forceinline__ uint64_t sort32(uint64_t k, int lane) {
#pragma unroll
    for (int size = 2; size < 32; size <<= 1)
#pragma unroll
        for (int j = size >> 1; j; j >>= 1) {
            const uint64_t o = __shfl_xor_sync(0xffffffffu, k, j);
            const bool up = (lane & size) != 0;  // every second run ascends
            k = ((lane & j) != 0) != up ? min64(k, o) : max64(k, o);
        }
    return order_bitonic(k, lane);
}
// b reversed against a: the larger of each pair are the best 32 of both, as a bitonic sequence.
__device__ __forceinline__ uint64_t merge32(uint64_t a, uint64_t b, int lane) {
    return order_bitonic(max64(a, __shfl_sync(0xffffffffu, b, 31 - lane)), lane);
}

// The block's candidates: everything pushed since the last selection and the best of before.
template <int T>
struct Candidates {
    static constexpr int kChunk = T * kVecs * 4;
    static constexpr int kKeep = 512;  // selection starts when more are held after a chunk
    uint64_t key[kKeep + kChunk];
    uint64_t list[T / 32][32];
    int count;
};

// Joins the warps' sorted lists in shared memory; every thread gets lane's entry of the best 32.
template <int T>
__device__ uint64_t join_lists(uint64_t mine, uint64_t (*list)[32], int warp, int lane) {
    __syncthreads();
    list[warp][lane] = mine;
#pragma unroll
    for (int n = T / 64; n; n >>= 1) {
        __syncthreads();
        if (warp < n) {
            mine = merge32(list[warp][lane], list[warp + n][lane], lane);
            __syncwarp();
            list[warp][lane] = mine;
        }
    }
    __syncthreads();
    return list[0][lane];
}

// The best 32 of the held candidates, sorted over the lanes of every warp.
template <int T>
__device__ uint64_t select_best(Candidates<T>& c, int warp, int lane) {
    const int n = c.count;
    uint64_t best = 0;
    for (int i = warp * 32; i < n; i += T) {
        const uint64_t k = i + lane < n ? c.key[i + lane] : 0;
        // (a batch with nothing above the list's last entry changes nothing)
        if (i < T || __any_sync(0xffffffffu, k > __shfl_sync(0xffffffffu, best, 31))) best = merge32(best, sort32(k, lane), lane);
    }
    return join_lists<T>(best, c.list, warp, lane);
}

// One cluster of `parts` CTAs of T threads per row; each streams its part of the row once, 16 logits a
// thread and chunk, the next chunk's loads issued before the present one is worked on.
//
// Bound by HBM (4 bytes a logit) while rows abound: about 8 instructions a logit against 25 that the
// SMs can issue in a logit's time.  Measured figures stand in the table of the design notes' section on
// these operators.
// Candidates: the k-th best of the first chunk's T per-thread maxima bounds the row's k-th best from
// below, so the first chunk pushes about k keys and later chunks k ln(n / chunk) in all; a chunk's
// elements are looked at one by one only where its maximum passes the bound.  The pushes' order does
// not matter: keys are distinct and the selection sorts them.
template <int T, bool TOP>
__global__ void __launch_bounds__(T, 1024 / T) logprobs_rows(float* __restrict__ logp, float* __restrict__ lse,
                                                             float* __restrict__ entropy, float* __restrict__ top_logp,
                                                             int32_t* __restrict__ top_id, const float* __restrict__ x,
                                                             const int32_t* __restrict__ id, int64_t cols, int64_t x_s1,
                                                             int top, int parts) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    Candidates<T>& cand = *(Candidates<T>*)smem_raw;
    __shared__ Part sh_part[T / 32];
    __shared__ Part peer_part[kMaxCluster];
    __shared__ uint64_t peer_list[TOP ? kMaxCluster : 1][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row = blockIdx.x / parts;
    const int rank = blockIdx.x % parts;
    if (parts > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    const float* p = x + row * x_s1;
    const int off = (int)((uintptr_t)p >> 2) & 3;
    const int64_t nvec = (off + cols + 3) >> 2, per = (nvec + parts - 1) / parts;
    const int64_t v0 = rank * per, v1 = min(v0 + per, nvec);
    if (TOP && threadIdx.x == 0) cand.count = 0;

    float m = -FLT_MAX, s = 0.0f, t = 0.0f;
    float bound = -INFINITY;  // later chunks push what is not at most this
    float4 next[kVecs];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int64_t vi = v0 + i * T + threadIdx.x;
        next[i] = load_logits(p, vi < v1 ? vi : nvec, nvec, off, cols);
    }
    for (int64_t base = v0; base < v1; base += T * kVecs) {
        float v[kVecs * 4];
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            v[4 * i] = next[i].x;
            v[4 * i + 1] = next[i].y;
            v[4 * i + 2] = next[i].z;
            v[4 * i + 3] = next[i].w;
        }
        if (base + T * kVecs < v1) {
#pragma unroll
            for (int i = 0; i < kVecs; ++i) {
                const int64_t vi = base + (kVecs + i) * T + threadIdx.x;
                next[i] = load_logits(p, vi < v1 ? vi : nvec, nvec, off, cols);
            }
        }
        float cm = v[0];
#pragma unroll
        for (int i = 1; i < kVecs * 4; ++i) cm = fmaxf(cm, v[i]);
        if (cm > m) {
            const float c = fmaxf(m - cm, kFar), e = exp2_fast(c * kLog2e);
            t = (t + c * s) * e;
            s *= e;
            m = cm;
        }
        float cs = 0.0f;
#pragma unroll
        for (int i = 0; i < kVecs * 4; ++i) {
            const float d = v[i] - m, e = exp2_fast(d * kLog2e);
            cs += e;
            t = fmaf(e, fmaxf(d, kFar), t);
        }
        s += cs;
        if (TOP) {
            // (columns of the chunk's elements; a NaN shows in cs)
            const int64_t c0 = (base + threadIdx.x) * 4 - off;
            bool over = false;
            if (base == v0) {
                uint64_t mine = 0;
#pragma unroll
                for (int i = 0; i < kVecs * 4; ++i) {
                    const int64_t c = c0 + (i >> 2) * (T * 4) + (i & 3);
                    if (c >= 0 && c < cols && base + (i >> 2) * T + threadIdx.x < v1) mine = max64(mine, rank_key(v[i], (uint32_t)c));
                }
                const uint64_t list = join_lists<T>(sort32(mine, lane), cand.list, warp, lane);
                const uint64_t least = __shfl_sync(0xffffffffu, list, top - 1);
                bound = key_value(least);
                if (bound != bound) bound = INFINITY;
                if (least == 0) bound = -INFINITY;
                if (mine >= least && mine) {
#pragma unroll
                    for (int i = 0; i < kVecs * 4; ++i) {
                        const int64_t c = c0 + (i >> 2) * (T * 4) + (i & 3);
                        if (c >= 0 && c < cols && base + (i >> 2) * T + threadIdx.x < v1) {
                            const uint64_t k = rank_key(v[i], (uint32_t)c);
                            if (k >= least) cand.key[atomicAdd(&cand.count, 1)] = k;
                        }
                    }
                }
            } else {
                if (!(cm <= bound) || cs != cs) {
#pragma unroll
                    for (int i = 0; i < kVecs * 4; ++i)
                        if (!(v[i] <= bound)) {  // (elements past the row are -inf)
                            const int at = atomicAdd(&cand.count, 1);
                            cand.key[at] = rank_key(v[i], (uint32_t)(c0 + (i >> 2) * (T * 4) + (i & 3)));
                            over |= at >= Candidates<T>::kKeep;
                        }
                }
                if (__syncthreads_or(over)) {
                    const uint64_t best = select_best<T>(cand, warp, lane);
                    if (warp == 0) {
                        cand.key[lane] = best;
                        if (lane == 0) cand.count = 32;
                    }
                    bound = key_value(__shfl_sync(0xffffffffu, best, top - 1));
                    if (bound != bound) bound = INFINITY;
                    __syncthreads();
                }
            }
        }
    }

    Part mine{m, (double)s, (double)t};
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const Part b{__shfl_xor_sync(0xffffffffu, mine.m, o), __shfl_xor_sync(0xffffffffu, mine.s, o),
                     __shfl_xor_sync(0xffffffffu, mine.t, o)};
        mine = join(mine, b);
    }
    if (lane == 0) sh_part[warp] = mine;
    __syncthreads();
    uint64_t list = 0;
    if (TOP) list = select_best<T>(cand, warp, lane);
    if (warp == 0) {
        mine = lane < T / 32 ? sh_part[lane] : Part{-FLT_MAX, 0.0, 0.0};
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            const Part b{__shfl_xor_sync(0xffffffffu, mine.m, o), __shfl_xor_sync(0xffffffffu, mine.s, o),
                         __shfl_xor_sync(0xffffffffu, mine.t, o)};
            mine = join(mine, b);
        }
    }
    if (parts > 1) {  // the parts meet in the first CTA, joined in their order
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // every CTA of the cluster runs
        cg::cluster_group cluster = cg::this_cluster();
        if (warp == 0) {
            if (lane == 0) *cluster.map_shared_rank(&peer_part[rank], 0) = mine;
            if (TOP) *cluster.map_shared_rank(&peer_list[rank][lane], 0) = list;
        }
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (rank) return;
        if (warp == 0) {
            mine = peer_part[0];
            for (int i = 1; i < parts; ++i) mine = join(mine, peer_part[i]);
            if (TOP)
                for (int i = 1; i < parts; ++i) list = merge32(list, peer_list[i][lane], lane);
        }
    }
    if (warp) return;
    const bool empty = mine.s == 0.0;  // nothing but -inf
    const double ln = empty ? -INFINITY : log(mine.s);
    if (lane == 0) {
        if (lse) lse[row] = empty ? -INFINITY : (float)((double)mine.m + ln);
        if (entropy) entropy[row] = empty ? 0.0f : (float)(ln - mine.t / mine.s);
        if (logp) {
            const int32_t i = id[row];
            logp[row] = i < 0 ? 0.0f : i >= cols ? __int_as_float(0x7FC00000) : empty ? -INFINITY : (float)((double)p[i] - mine.m - ln);
        }
    }
    if (TOP && lane < top) {
        if (top_id) top_id[row * top + lane] = (int32_t)(0xFFFFFFFFu - (uint32_t)list);
        if (top_logp) top_logp[row * top + lane] = empty ? -INFINITY : (float)((double)key_value(list) - mine.m - ln);
    }
}

// Four vectors a thread of one row's chunk; bound by HBM (8 bytes a logit).
constexpr int kBackThreads = 256;
constexpr int kBackVecs = 4;

__global__ void __launch_bounds__(kBackThreads) logprobs_backward(float* dx, const float* x, const int32_t* __restrict__ id,
                                                                  const float* __restrict__ lse,
                                                                  const float* __restrict__ entropy,
                                                                  const float* __restrict__ g_logp,
                                                                  const float* __restrict__ g_entropy, int64_t cols,
                                                                  int64_t x_s1, int64_t dx_s1, int64_t chunks) {
    const int64_t row = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
    const float* p = x + row * x_s1;
    float* q = dx + row * dx_s1;
    const float l = lse[row];
    const bool none = l == -INFINITY;
    const int32_t hot = g_logp ? id[row] : -1;
    const float g = hot < 0 || none ? 0.0f : hot >= cols ? __int_as_float(0x7FC00000) : g_logp[row];
    const float ge = g_entropy ? g_entropy[row] : 0.0f, en = g_entropy ? entropy[row] : 0.0f;
    const auto grad = [&](float v, int64_t c) {
        const float d = v - l, e = exp2_fast(d * kLog2e);
        const float r = -e * fmaf(ge, fmaxf(d, kFar) + en, g);
        return none ? 0.0f : c == hot ? r + g : r;
    };
    const int off = (int)((uintptr_t)p >> 2) & 3;
    const bool vec = ((((uintptr_t)p) ^ ((uintptr_t)q)) & 15) == 0;
    float4 v[kBackVecs];
#pragma unroll
    for (int i = 0; i < kBackVecs; ++i) {
        const int64_t c = ((chunk * kBackVecs + i) * kBackThreads + threadIdx.x) * 4 - off;
        if (vec && c >= 0 && c + 4 <= cols) v[i] = __ldcs((const float4*)(p + c));
    }
#pragma unroll
    for (int i = 0; i < kBackVecs; ++i) {
        const int64_t c = ((chunk * kBackVecs + i) * kBackThreads + threadIdx.x) * 4 - off;
        if (vec && c >= 0 && c + 4 <= cols) {
            __stcs((float4*)(q + c), make_float4(grad(v[i].x, c), grad(v[i].y, c + 1), grad(v[i].z, c + 2), grad(v[i].w, c + 3)));
        } else {
            for (int j = 0; j < 4; ++j)
                if (c + j >= 0 && c + j < cols) q[c + j] = grad(p[c + j], c + j);
        }
    }
}

template <int T, bool TOP>
int run_rows(float* logp, float* lse, float* entropy, float* top_logp, int32_t* top_id, const float* x, const int32_t* id,
             int64_t rows, int64_t cols, int64_t x_s1, int top, int parts, cudaStream_t st) {
    const int smem = TOP ? (int)sizeof(Candidates<T>) : 0;
    const auto kern = logprobs_rows<T, TOP>;
    if (smem) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return (int)e;
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)parts;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(rows * parts));
    cfg.blockDim = dim3(T);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = parts > 1 ? 1 : 0;
    return (int)cudaLaunchKernelEx(&cfg, kern, logp, lse, entropy, top_logp, top_id, x, id, cols, x_s1, top, parts);
}

}  // namespace

extern "C" int mcu_launch_logprobs(float* logp, float* lse, float* entropy, float* top_logp, int32_t* top_id,
                                   const float* x, const int32_t* id, int64_t rows, int64_t cols, int64_t x_s1, int top,
                                   cudaStream_t st, int* launches) {
    *launches = 1;
    if (cols <= 4096)  // short rows: small blocks
        return top ? run_rows<128, true>(logp, lse, entropy, top_logp, top_id, x, id, rows, cols, x_s1, top, 1, st)
                   : run_rows<128, false>(logp, lse, entropy, top_logp, top_id, x, id, rows, cols, x_s1, top, 1, st);
    int parts = 1;  // few rows: up to 8 CTAs share one, at least a chunk of 8192 logits each
    while (parts < kMaxCluster && rows * parts < 148 && cols >= 2 * 8192 * (int64_t)parts) parts *= 2;
    return top ? run_rows<512, true>(logp, lse, entropy, top_logp, top_id, x, id, rows, cols, x_s1, top, parts, st)
               : run_rows<512, false>(logp, lse, entropy, top_logp, top_id, x, id, rows, cols, x_s1, top, parts, st);
}

extern "C" int mcu_launch_logprobs_backward(float* dx, const float* x, const int32_t* id, const float* lse,
                                            const float* entropy, const float* g_logp, const float* g_entropy,
                                            int64_t rows, int64_t cols, int64_t x_s1, int64_t dx_s1, cudaStream_t st,
                                            int* launches) {
    const int64_t chunks = (cols + 3 + kBackThreads * kBackVecs * 4 - 1) / (kBackThreads * kBackVecs * 4);
    if (rows * chunks > 0x7fffffff) return (int)cudaErrorInvalidValue;
    logprobs_backward<<<(unsigned)(rows * chunks), kBackThreads, 0, st>>>(dx, x, id, lse, entropy, g_logp, g_entropy, cols,
                                                                          x_s1, dx_s1, chunks);
    *launches = 1;
    return (int)cudaGetLastError();
}
