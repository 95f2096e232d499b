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
#include <type_traits>
#include "mcu_kernels.h"
#include "mcu_launch.cuh"
#include "mcu_lm.cuh"

namespace cg = cooperative_groups;
using namespace mcu;

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFar = -1e30f;  // stands for d = -inf where it meets a factor of zero
constexpr int kVecs = 4;        // float4 per thread and chunk
constexpr int kMaxCluster = 8;  // CTAs that share a row
constexpr int kSms = 148;

__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// The order of logits as an integer (NaN above everything, -0 as +0), and with the column below it, so
// that of equal logits the lower column comes first.  0 stands for no element.
__device__ __forceinline__ uint32_t order_of(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return v != v ? 0xFFFFFFFFu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t rank_key(uint32_t order, uint32_t col) { return (uint64_t)order << 32 | (0xFFFFFFFFu - col); }
constexpr uint32_t kOrderInf = 0xFF800000u;  // of +inf
__device__ __forceinline__ float order_value(uint32_t b) { return __uint_as_float((b & 0x80000000u) ? b & 0x7FFFFFFFu : ~b); }
__device__ __forceinline__ float key_value(uint64_t key) { return order_value((uint32_t)(key >> 32)); }

// A row whose first logit lies `off` floats past a 16-byte boundary, as vectors of four: vector vi holds
// the elements 4 vi - off .. + 3.  Only the first and the last one may reach past the row; their elements
// there are -inf, and nothing outside the row is read.
struct Row {
    const float* p;
    int64_t cols;
    int off;
    int full0, full1;  // vectors that lie inside the row
};
__device__ __forceinline__ Row row_of(const float* p, int64_t cols) {
    const int off = (int)((uintptr_t)p >> 2) & 3;
    return Row{p, cols, off, off ? 1 : 0, (int)((off + cols) >> 2)};
}
__device__ __forceinline__ int vectors_of(const Row& r) { return (int)((r.off + r.cols + 3) >> 2); }
__device__ __noinline__ float4 load_edge(const float* p, int64_t cols, int64_t c) {
    float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    if (c >= 0 && c < cols) v.x = p[c];
    if (c + 1 >= 0 && c + 1 < cols) v.y = p[c + 1];
    if (c + 2 >= 0 && c + 2 < cols) v.z = p[c + 2];
    if (c + 3 >= 0 && c + 3 < cols) v.w = p[c + 3];
    return v;
}
// The thread's kVecs vectors of the chunk of T * kVecs at `base`, those from v1 on as -inf.
template <int T>
__device__ __forceinline__ void load_chunk(float4 (&v)[kVecs], const Row& r, int base, int v1) {
    const int first = base + (int)threadIdx.x;
    const float4* q = (const float4*)(r.p - r.off) + first;
    if (base >= r.full0 && base + T * kVecs <= min(r.full1, v1)) {
#pragma unroll
        for (int i = 0; i < kVecs; ++i) v[i] = __ldcs(q + i * T);
        return;
    }
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int vi = first + i * T;
        if (vi >= v1) v[i] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        else if (vi >= r.full0 && vi < r.full1) v[i] = __ldcs(q + i * T);
        else v[i] = load_edge(r.p, r.cols, (int64_t)vi * 4 - r.off);
    }
}

struct Part {
    float m;
    double s, t;
};
// A warp's parts as one, on every lane: all are brought to the largest maximum, then added.  (A part of
// nothing has s = t = 0 and the lowest maximum; the bounded distance keeps 0 * distance at 0.)
__device__ __forceinline__ Part join_warp(Part a) {
    float m = a.m;
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float c = fmaxf(a.m - m, kFar);
    const double e = (double)expf(c);
    a.t = (a.t + (double)c * a.s) * e;
    a.s *= e;
    a.m = m;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
        a.t += __shfl_xor_sync(0xffffffffu, a.t, o);
    }
    return a;
}

// Bitonic networks over a warp's lanes, descending; K is a 32-bit order or a 64-bit key.
template <typename K>
__device__ __forceinline__ K order_bitonic(K k, int lane) {
#pragma unroll
    for (int j = 16; j; j >>= 1) {
        const K o = __shfl_xor_sync(0xffffffffu, k, j);
        k = ((lane & j) != 0) == (k > o) ? o : k;
    }
    return k;
}
template <typename K>
__device__ __forceinline__ K sort32(K k, int lane) {
#pragma unroll
    for (int size = 2; size < 32; size <<= 1)
#pragma unroll
        for (int j = size >> 1; j; j >>= 1) {
            const K o = __shfl_xor_sync(0xffffffffu, k, j);
            // every second run ascends
            k = (((lane & j) != 0) != ((lane & size) != 0)) == (k > o) ? o : k;
        }
    return order_bitonic(k, lane);
}
// b reversed against a: the larger of each pair are the best 32 of both, as a bitonic sequence.
template <typename K>
__device__ __forceinline__ K merge32(K a, K b, int lane) {
    b = __shfl_sync(0xffffffffu, b, 31 - lane);
    return order_bitonic(a > b ? a : b, lane);
}

// The candidates of a block: each warp fills a buffer of its own without asking the others, cut down to
// its best 32 when a chunk leaves more than kKeep; at the end the warps' rests meet in the pool.
constexpr int kKeep = 64;
template <int T>
struct Candidates {
    static constexpr int kWarps = T / 32;
    uint64_t key[kWarps][kKeep + 32 * kVecs * 4];
    uint64_t pool[kWarps * kKeep];
    uint64_t list[kWarps][32];
    uint32_t group[64];  // maxima of 64 groups of threads over the first chunk
    uint32_t first;      // the bound that the groups gave
    uint32_t least;      // the bound that full buffers gave
    int pooled;
};

// The best 32 of n keys, sorted over the lanes of the calling warp.
__device__ __noinline__ uint64_t best_of(const uint64_t* key, int n, int lane) {
    uint64_t best = 0;
    for (int i = 0; i < n; i += 32) {
        const uint64_t k = i + lane < n ? key[i + lane] : 0;
        // (a batch with nothing above the list's last entry changes nothing)
        if (!i) best = sort32(k, lane);
        else if (__any_sync(0xffffffffu, k > __shfl_sync(0xffffffffu, best, 31))) best = merge32(best, sort32(k, lane), lane);
    }
    return best;
}

// The top-th largest maximum of 64 groups of threads, from each thread's; 0 if fewer have one.
template <int T>
__device__ __forceinline__ uint32_t group_bound(Candidates<T>& cand, uint32_t big, int top, int warp, int lane) {
#pragma unroll
    for (int o = 1; o < T / 64; o <<= 1) big = max(big, __shfl_xor_sync(0xffffffffu, big, o));
    if (threadIdx.x % (T / 64) == 0) cand.group[threadIdx.x / (T / 64)] = big;
    __syncthreads();
    if (warp == 0) {
        const uint32_t list = merge32(sort32(cand.group[lane], lane), sort32(cand.group[lane + 32], lane), lane);
        const uint32_t least = __shfl_sync(0xffffffffu, list, top - 1);
        if (lane == 0) cand.first = least;
    }
    __syncthreads();
    return cand.first;
}

// One cluster of `parts` CTAs of T threads per row; each streams its part of the row once, 16 logits a
// thread and chunk, the next chunk's loads issued before the present one is worked on.  Bound by HBM, 4
// bytes a logit: 4095 x 100003 takes 247 us without alternatives (6.6 TB/s) and 298 us with 8 of them (5.5),
// the rest being the bound's barriers, the chunks in which a candidate shows and, for rows of few chunks, misses of
// the instruction cache (8192 x 4096: 29 us without alternatives, 67 with five).  Collecting candidates for
// the whole block, with a barrier a chunk, took 520 us.
//
// Candidates: the top-th largest of 64 group maxima of the first chunk is a lower bound of the row's top-th
// logit, so that little more than `top` of the first chunk's logits pass it, as many in each later chunk,
// and from the fifth on, with the maxima of four, a quarter of that: a warp looks at single elements only
// where the maximum of a lane's 16 passes, and then where that of four does.  Later elements have higher
// columns than the at least `top` that reached the bound, so they have to exceed it; a bound that a warp's
// full buffer gives has to be reached only, since another warp may still be at lower columns.  The order in
// which candidates are found does not matter: keys are distinct and sorted at the end.
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
    pdl_begin();
    const Row r = row_of(x + row * x_s1, cols);
    const int nvec = vectors_of(r), per = (nvec + parts - 1) / parts;
    const int v0 = min(rank * per, nvec), v1 = min(v0 + per, nvec);
    if (TOP && threadIdx.x == 0) cand.pooled = 0, cand.least = 0;  // (seen by all after the first chunk's barriers)

    float m = -FLT_MAX, s = 0.0f, t = 0.0f;
    int held = 0;         // keys in this warp's buffer
    uint32_t exceed = 0;  // the least order of a candidate after the first chunk
    float4 next[kVecs];
    load_chunk<T>(next, r, v0, v1);
    for (int base = v0; base < v1; base += T * kVecs) {
        float v[kVecs * 4];
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            v[4 * i] = next[i].x;
            v[4 * i + 1] = next[i].y;
            v[4 * i + 2] = next[i].z;
            v[4 * i + 3] = next[i].w;
        }
        if (base + T * kVecs < v1) load_chunk<T>(next, r, base + T * kVecs, v1);
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
        if constexpr (TOP) {
            const uint32_t c0 = (uint32_t)(base + (int)threadIdx.x) * 4 - r.off;  // column of v[0]
            const auto push = [&](bool yes, float value, int i) {
                const uint32_t who = __ballot_sync(0xffffffffu, yes);
                if (yes)
                    cand.key[warp][held + __popc(who & ((1u << lane) - 1))] =
                        rank_key(order_of(value), c0 + (i >> 2) * (T * 4) + (i & 3));
                held += __popc(who);
            };
            if (base == v0) {
                // bit i: element i is one of the part's (not so past an edge of the row or the part)
                uint32_t inside = 0xFFFF;
                if (base < r.full0 || base + T * kVecs > min(r.full1, v1)) {
                    inside = 0;
#pragma unroll
                    for (int i = 0; i < kVecs * 4; ++i) {
                        const int vi = base + (i >> 2) * T + (int)threadIdx.x;
                        const int64_t c = (int64_t)vi * 4 - r.off + (i & 3);
                        inside |= (vi < v1 && c >= 0 && c < cols ? 1u : 0u) << i;
                    }
                }
                uint32_t big = inside == 0xFFFF && cs == cs ? order_of(cm) : 0;
                if (inside != 0xFFFF || cs != cs) {
#pragma unroll
                    for (int i = 0; i < kVecs * 4; ++i)
                        if (inside >> i & 1) big = max(big, order_of(v[i]));
                }
                const uint32_t least = group_bound<T>(cand, big, top, warp, lane);
                if (__any_sync(0xffffffffu, big >= least)) {
#pragma unroll
                    for (int q = 0; q < kVecs * 4; q += 4) {
                        const float top4 = fmaxf(fmaxf(v[q], v[q + 1]), fmaxf(v[q + 2], v[q + 3]));
                        if (!__any_sync(0xffffffffu, order_of(top4) >= least || cs != cs)) continue;
#pragma unroll
                        for (int i = q; i < q + 4; ++i) {
                            const bool yes = (inside >> i & 1) && order_of(v[i]) >= least;
                            if (__any_sync(0xffffffffu, yes)) push(yes, v[i], i);
                        }
                    }
                }
                exceed = least + (least < kOrderInf);
            } else {
                // as a logit, so that one comparison finds candidates and NaN; +inf where only NaN are above
                const float least = order_value(min(max(exceed, *(volatile uint32_t*)&cand.least), kOrderInf));
                if (__any_sync(0xffffffffu, !(cm < least) || cs != cs)) {
#pragma unroll
                    for (int q = 0; q < kVecs * 4; q += 4) {  // (elements past the row are -inf, below any bound here)
                        const float top4 = fmaxf(fmaxf(v[q], v[q + 1]), fmaxf(v[q + 2], v[q + 3]));
                        if (!__any_sync(0xffffffffu, !(top4 < least) || cs != cs)) continue;
#pragma unroll
                        for (int i = q; i < q + 4; ++i) {
                            const bool yes = !(v[i] < least);
                            if (__any_sync(0xffffffffu, yes)) push(yes, v[i], i);
                        }
                    }
                }
            }
            // four chunks on, the running maxima give a bound four times as sharp
            if (base - v0 == 3 * T * kVecs && v1 - base > 4 * T * kVecs) {
                const uint32_t least = group_bound<T>(cand, order_of(m), top, warp, lane);
                // (the lowest value is also the maximum of a thread that has seen nothing above -inf)
                if (least > order_of(-FLT_MAX)) exceed = max(exceed, least + (least < kOrderInf));
            }
            if (held > kKeep) {
                __syncwarp();
                const uint64_t best = best_of(cand.key[warp], held, lane);
                __syncwarp();
                cand.key[warp][lane] = best;
                held = 32;
                const uint32_t o = (uint32_t)(__shfl_sync(0xffffffffu, best, top - 1) >> 32);
                if (lane == 0) atomicMax(&cand.least, o);
                __syncwarp();
            }
        }
    }

    Part mine = join_warp(Part{m, (double)s, (double)t});
    if (lane == 0) sh_part[warp] = mine;
    uint64_t list = 0;
    if constexpr (TOP) {
        __syncwarp();
        int at = 0;
        if (lane == 0 && held) at = atomicAdd(&cand.pooled, held);
        at = __shfl_sync(0xffffffffu, at, 0);
        for (int i = lane; i < held; i += 32) cand.pool[at + i] = cand.key[warp][i];
        __syncthreads();
        const int n = cand.pooled;
        const bool count = T == 512 && n <= 128;
        const int lists = count ? 0 : (n + 31) / 32;  // a list per 32 keys
        if (count) {
            // where latency counts a key's place is the number of larger ones (no two are equal), which is no chain
            // of exchanges (4 x 131072: 9.5 us, 9.9); it takes more instructions, which small blocks have no room for
            if (warp * 32 < n) {
                const int i = warp * 32 + lane;
                const uint64_t k = i < n ? cand.pool[i] : 0;
                int place = 0;
#pragma unroll 8
                for (int j = 0; j < n; ++j) place += cand.pool[j] > k;
                if (i < n && place < 32) cand.list[0][place] = k;
            }
            if (n > 32) __syncthreads();
            else __syncwarp();
            if (warp == 0 && lane < n) list = cand.list[0][lane];
        } else if (warp < lists) {
            for (int i = warp * 32; i < n; i += T) {
                const uint64_t k = sort32(i + lane < n ? cand.pool[i + lane] : 0, lane);
                list = i == warp * 32 ? k : merge32(list, k, lane);
            }
            cand.list[warp][lane] = list;
        }
        for (int k = min(lists, T / 32); k > 1; k = (k + 1) / 2) {  // the upper half of the lists into the lower
            __syncthreads();
            const int h = (k + 1) / 2;
            if (warp + h < k) {
                list = merge32(list, cand.list[warp + h][lane], lane);
                cand.list[warp][lane] = list;
            }
        }
    } else {
        __syncthreads();
    }
    if (warp == 0) mine = join_warp(lane < T / 32 ? sh_part[lane] : Part{-FLT_MAX, 0.0, 0.0});
    if (parts > 1) {  // the parts meet in the first CTA
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // every CTA of the cluster runs
        cg::cluster_group cluster = cg::this_cluster();
        if (warp == 0) {
            if (lane == 0) *cluster.map_shared_rank(&peer_part[rank], 0) = mine;
            if (TOP) *cluster.map_shared_rank(&peer_list[rank][lane], 0) = list;
        }
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (rank) return;
        if constexpr (TOP) {
            if (warp < parts) list = peer_list[warp][lane];
            for (int k = parts; k > 1; k = (k + 1) / 2) {
                const int h = (k + 1) / 2;
                if (warp + h < k) {
                    list = merge32(list, peer_list[warp + h][lane], lane);
                    peer_list[warp][lane] = list;
                }
                __syncthreads();
            }
        }
        if (warp == 0) mine = join_warp(lane < parts ? peer_part[lane] : Part{-FLT_MAX, 0.0, 0.0});
    }
    if (warp) return;
    const bool empty = mine.s == 0.0;  // nothing but -inf
    const double ln = empty ? -INFINITY : log(mine.s);
    if (lane == 0) {
        if (lse) lse[row] = empty ? -INFINITY : (float)((double)mine.m + ln);
        if (entropy) entropy[row] = empty ? 0.0f : (float)(ln - mine.t / mine.s);
        if (logp) {
            const int32_t i = id[row];
            logp[row] = i < 0 ? 0.0f : i >= cols ? __int_as_float(0x7FC00000) : empty ? -INFINITY : (float)((double)r.p[i] - mine.m - ln);
        }
    }
    if (TOP && lane < top) {
        if (top_id) top_id[row * top + lane] = (int32_t)(0xFFFFFFFFu - (uint32_t)list);
        if (top_logp) top_logp[row * top + lane] = empty ? -INFINITY : (float)((double)key_value(list) - mine.m - ln);
    }
}

// Four vectors a thread of one row's chunk; bound by HBM, 8 bytes a logit (2048 x 65600: 168 us, 6.4 TB/s).
constexpr int kBackThreads = 256;
constexpr int kBackVecs = 4;
// The least log probability that counts: e^d is 0 in f32 from -104 on, and 0 times a distance bounded here is 0 for
// gradients of the entropy up to 2^120 (with kFar for a bound it was 0 times infinity from 3.4e8 on).
constexpr float kGone = -128.0f;

__global__ void __launch_bounds__(kBackThreads) logprobs_backward(float* dx, const float* x, const int32_t* __restrict__ id,
                                                                  const float* __restrict__ lse,
                                                                  const float* __restrict__ entropy,
                                                                  const float* __restrict__ g_logp,
                                                                  const float* __restrict__ g_entropy, int64_t cols,
                                                                  int64_t x_s1, int64_t dx_s1, int64_t chunks) {
    pdl_begin();
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
        const float r = -e * fmaf(ge, fmaxf(d, kGone) + en, g);
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
        static bool done[64];
        cudaError_t e = allow_smem(kern, smem, done);
        if (e != cudaSuccess) return (int)e;
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)parts;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(rows * parts));
    cfg.blockDim = dim3(T);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = parts > 1 ? 2 : 1;
    return (int)cudaLaunchKernelEx(&cfg, kern, logp, lse, entropy, top_logp, top_id, x, id, cols, x_s1, top, parts);
}

}  // namespace

extern "C" int mcu_launch_logprobs(float* logp, float* lse, float* entropy, float* top_logp, int32_t* top_id,
                                   const float* x, const int32_t* id, int64_t rows, int64_t cols, int64_t x_s1, int top,
                                   cudaStream_t st, int* launches) {
    *launches = 1;
    const auto go = [&](auto threads, int parts) {
        constexpr int T = decltype(threads)::value;
        return top ? run_rows<T, true>(logp, lse, entropy, top_logp, top_id, x, id, rows, cols, x_s1, top, parts, st)
                   : run_rows<T, false>(logp, lse, entropy, top_logp, top_id, x, id, rows, cols, x_s1, top, parts, st);
    };
    // Few rows: blocks of 512 threads, two an SM, up to 8 of them sharing a row of at least two chunks of 8192
    // logits each, or eight where they share an SM (148 x 131072 with 20 alternatives: 21.0 us with two parts,
    // 22.9 with one, 34 with 256 threads; 100 x 32000: 11.0 with one, 12.1 with two).
    // Many: an SM's 1024 threads as small blocks, whose barriers and ends overlap better, yet not so small
    // that the first chunk says little about the row: on the device 4095 x 100003 with 8 alternatives takes 311, 289
    // and 354 us with 512, 256 and 128 threads, 8192 x 5000 with 5 takes 192, 106 and 78 us, 8192 x 20000 with 20
    // takes 209 and 179 us with 256 and 128, 8192 x 32000 248 and 231, 4096 x 50257 175 and 200.  Long rows
    // whose last wave would be short take the larger blocks (700 x 131072: 73 us, 82).
    const auto waves = [&](int64_t blocks) { return (rows + kSms * blocks - 1) / (kSms * blocks); };  // of so many blocks an SM
    if (rows <= 2 * kSms && cols > (rows <= kSms ? 8192 : 16384)) {
        int parts = 1;
        while (parts < kMaxCluster && rows * parts <= kSms && cols >= (rows * parts * 2 <= kSms ? 2 : 8) * 8192 * (int64_t)parts) parts *= 2;
        return go(std::integral_constant<int, 512>(), parts);
    }
    if (cols > 65536 && waves(2) * 4 <= waves(4) * 2 * 3) return go(std::integral_constant<int, 512>(), 1);
    if (cols > (waves(8) > 1 ? 32768 : 8192) || (rows <= 2 * kSms && cols > 2048)) return go(std::integral_constant<int, 256>(), 1);
    return go(std::integral_constant<int, 128>(), 1);
}

extern "C" int mcu_launch_logprobs_backward(float* dx, const float* x, const int32_t* id, const float* lse,
                                            const float* entropy, const float* g_logp, const float* g_entropy,
                                            int64_t rows, int64_t cols, int64_t x_s1, int64_t dx_s1, cudaStream_t st,
                                            int* launches) {
    const int64_t chunks = (cols + 3 + kBackThreads * kBackVecs * 4 - 1) / (kBackThreads * kBackVecs * 4);
    if (rows * chunks > 0x7fffffff) return (int)cudaErrorInvalidValue;
    *launches = 1;
    return (int)launch_dep(logprobs_backward, dim3((unsigned)(rows * chunks)), dim3(kBackThreads), 0, st, dx, x, id, lse, entropy,
                           g_logp, g_entropy, cols, x_s1, dx_s1, chunks);
}
