// k_heads.cu - head norm and position rotation (mag_cuda_rotate_heads_f32 and its gradient), and the paged cache's write
// and read (mag_cuda_kv_write, mag_cuda_kv_read).
#include <cuda_runtime.h>
#include <cstdint>
#include "mcu_kernels.h"
#include "mcu_launch.cuh"
#include "mcu_lm.cuh"

using namespace mcu;

namespace {

// A head row of dim values lies in the registers of a group of LANES lanes of a warp: lane l holds the chunks
// l + LANES v of four values each, v < V.  All of a norm's and a rotation's exchange is then shuffles within the group.
// Groups of 16 lanes hold heads of up to 64 values, two to a warp.
constexpr int kHeadThreads = 256, kHeadWarps = 8;
constexpr int kMaxPairs = 128;

template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
template <int LANES>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

template <bool VEC>
__device__ __forceinline__ float4 load4(const float* p) {
    if (VEC) return *(const float4*)p;
    return make_float4(p[0], p[1], p[2], p[3]);
}
template <bool VEC>
__device__ __forceinline__ void store4(float* p, float4 v) {
    if (VEC) {
        *(float4*)p = v;
    } else {
        p[0] = v.x, p[1] = v.y, p[2] = v.z, p[3] = v.w;
    }
}

// (cos, sin) of pos * f, times mag.  The angle is formed in f64 and reduced there to n quarter turns and |r| <= pi / 4
// (pi / 2 as a sum of two f64); what r loses as an f32 is put back to first order, so that the results are within about
// an f32 rounding for every int32 position.
__device__ __forceinline__ float2 turn_of(int pos, float f, float mag) {
    const double a = (double)pos * (double)f, n = rint(a * 0.63661977236758134);
    const double r = fma(-n, 6.123233995736766e-17, fma(-n, 1.5707963267948966, a));
    const float rf = (float)r, dr = (float)(r - (double)rf);
    float s, c;
    sincosf(rf, &s, &c);
    const float sn = fmaf(dr, c, s), cn = fmaf(-dr, s, c);
    const int q = (int)((long long)n & 3);
    const float cq = q == 0 ? cn : q == 1 ? -sn : q == 2 ? -cn : sn, sq = q == 0 ? sn : q == 1 ? cn : q == 2 ? -sn : -cn;
    return make_float2(cq * mag, sq * mag);
}

struct Turn {
    const int32_t* pos;
    const float* freq;
    int rot, pairs;  // pairs: neighbouring values turn together, else the two halves of the rotated part
    float mag;
};

// This lane's factors of one token's turn, from the token's cosines and sines: y = x c + partner s.
template <int LANES, int V>
__device__ __forceinline__ void turn_factors(float (&c)[4 * V], float (&s)[4 * V], const float* cs, const float* sn, const Turn& t, int l,
                                             bool back) {
    const float sign = back ? -1.0f : 1.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int d = 4 * (l + LANES * v);
        if (d >= t.rot) continue;
        if (t.pairs) {
            const float2 a = *(const float2*)(cs + d / 2), b = *(const float2*)(sn + d / 2);
            c[4 * v] = c[4 * v + 1] = a.x, c[4 * v + 2] = c[4 * v + 3] = a.y;
            s[4 * v] = -sign * b.x, s[4 * v + 1] = sign * b.x, s[4 * v + 2] = -sign * b.y, s[4 * v + 3] = sign * b.y;
        } else {
            const int half = t.rot / 2, p = d < half ? d : d - half;
            const float4 a = *(const float4*)(cs + p), b = *(const float4*)(sn + p);
            const float g = d < half ? -sign : sign;
            c[4 * v] = a.x, c[4 * v + 1] = a.y, c[4 * v + 2] = a.z, c[4 * v + 3] = a.w;
            s[4 * v] = g * b.x, s[4 * v + 1] = g * b.y, s[4 * v + 2] = g * b.z, s[4 * v + 3] = g * b.w;
        }
    }
}
// x turned; chunks behind the rotated part stay bit for bit.  All lanes of the warp take part.
template <int LANES, int V>
__device__ __forceinline__ void turn(float (&x)[4 * V], const float (&c)[4 * V], const float (&s)[4 * V], const Turn& t, int l) {
    float o[4 * V];
    if (t.pairs) {
#pragma unroll
        for (int i = 0; i < 4 * V; ++i) o[i] = x[i ^ 1];
    } else {
        const int shift = t.rot / 8;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int k = l + LANES * v, m = 4 * k < t.rot / 2 ? k + shift : k - shift;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float a = __shfl_sync(0xffffffffu, x[i], m & (LANES - 1), LANES);
                if (V == 2) {
                    const float b = __shfl_sync(0xffffffffu, x[4 * (V - 1) + i], m & (LANES - 1), LANES);
                    a = m >= LANES ? b : a;
                }
                o[4 * v + i] = a;
            }
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
        if (4 * (l + LANES * v) < t.rot) {
#pragma unroll
            for (int i = 4 * v; i < 4 * v + 4; ++i) x[i] = fmaf(x[i], c[i], o[i] * s[i]);
        }
}

// ------------------------------------------------------------ forward and cache write
//
// One block serves one token (blockIdx.x) and up to 8 warps x U head rows of each group: first the loads of all of them,
// then the token's cosines and sines, once for the block, under the loads' latency, then the rows.  Query rows go out in
// f32, key and value rows as e4m3 with their scale.
// What bounds it: HBM, one read and one write of each value.
struct HeadArgs {
    const float *q, *k, *v, *q_w, *k_w;
    float *q_out, *rstd;
    uint8_t *kq, *vq;
    float *ks, *vs;
    const int32_t* slot;
    Turn turn;
    float eps;
    int dim, q_heads, heads, page_log, slots;  // heads: of keys and of values, 0 without a cache
    int64_t q_s1, k_s1, v_s1, out_s1;
};

template <int LANES, int V, int U, bool VEC>
__global__ void __launch_bounds__(kHeadThreads) heads_forward(HeadArgs a) {
    __shared__ __align__(16) float cs[kMaxPairs], sn[kMaxPairs];
    constexpr int GROUPS = kHeadWarps * 32 / LANES;
    const int l = threadIdx.x & (LANES - 1), group = threadIdx.x / LANES;
    const int64_t row = blockIdx.x;
    const int jobs = a.q_heads + 2 * a.heads;
    pdl_begin();
    float x[U][4 * V];
    int job[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        int j = ((int)blockIdx.y * U + u) * GROUPS + group;
        const float* p = nullptr;
        if (j < a.q_heads) {
            p = a.q + row * a.q_s1 + (int64_t)j * a.dim;
        } else if (j < a.q_heads + a.heads) {
            p = a.k + row * a.k_s1 + (int64_t)(j - a.q_heads) * a.dim;
        } else if (j < jobs) {
            p = a.v + row * a.v_s1 + (int64_t)(j - a.q_heads - a.heads) * a.dim;
        }
        job[u] = p ? j : -1;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int d = 4 * (l + LANES * v);
            float4 t = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (p && d < a.dim) t = load4<VEC>(p + d);
            x[u][4 * v] = t.x, x[u][4 * v + 1] = t.y, x[u][4 * v + 2] = t.z, x[u][4 * v + 3] = t.w;
        }
    }
    const int slot = a.heads ? a.slot[row] : -1;
    if (a.turn.rot) {
        const int pos = a.turn.pos[row];
        for (int i = threadIdx.x; i < a.turn.rot / 2; i += kHeadThreads) {
            const float2 t = turn_of(pos, a.turn.freq[i], a.turn.mag);
            cs[i] = t.x, sn[i] = t.y;
        }
        __syncthreads();
    }
    float c[4 * V] = {}, s[4 * V] = {};
    turn_factors<LANES, V>(c, s, cs, sn, a.turn, l, false);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int j = job[u];
        const bool query = j >= 0 && j < a.q_heads, value = j >= a.q_heads + a.heads;
        const float* w = query ? a.q_w : value ? nullptr : a.k_w;
        if (a.q_w || a.k_w) {
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < 4 * V; ++i) ss = fmaf(x[u][i], x[u][i], ss);
            const float r = inv_sqrt(group_sum<LANES>(ss) / (float)a.dim + a.eps);
            if (w) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const int d = 4 * (l + LANES * v);
                    if (d < a.dim) {
                        const float4 t = load4<VEC>(w + d);
                        x[u][4 * v] = x[u][4 * v] * r * t.x, x[u][4 * v + 1] = x[u][4 * v + 1] * r * t.y;
                        x[u][4 * v + 2] = x[u][4 * v + 2] * r * t.z, x[u][4 * v + 3] = x[u][4 * v + 3] * r * t.w;
                    }
                }
                if (query && a.rstd && l == 0) a.rstd[row * a.q_heads + j] = r;
            }
        }
        if (a.turn.rot) {
            float y[4 * V];
#pragma unroll
            for (int i = 0; i < 4 * V; ++i) y[i] = x[u][i];
            turn<LANES, V>(y, c, s, a.turn, l);
#pragma unroll
            for (int i = 0; i < 4 * V; ++i) x[u][i] = value ? x[u][i] : y[i];
        }
        if (query) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int d = 4 * (l + LANES * v);
                if (d < a.dim)
                    store4<VEC>(a.q_out + row * a.out_s1 + (int64_t)j * a.dim + d,
                                make_float4(x[u][4 * v], x[u][4 * v + 1], x[u][4 * v + 2], x[u][4 * v + 3]));
            }
        }
        if (V == 1 && a.heads) {  // (a cache's heads have at most 128 values)
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) top = max(top, abs_bits(x[u][i]));
            top = group_max<LANES>(top);
            if (j >= a.q_heads && (uint32_t)slot < (uint32_t)a.slots) {
                const int h = j - a.q_heads - (value ? a.heads : 0);
                const int64_t at = ((((int64_t)(slot >> a.page_log) * a.heads) + h) << a.page_log) + (slot & ((1 << a.page_log) - 1));
                const E4m3Group g = e4m3_group(top);
                const bool bad = top >= 0x7F800000u;
                if (4 * l < a.dim)
                    *(uint32_t*)((value ? a.vq : a.kq) + at * a.dim + 4 * l) =
                        bad ? 0u : e4m3_quotients(g, x[u][0], x[u][1], x[u][2], x[u][3]);
                if (l == 0) (value ? a.vs : a.ks)[at] = bad ? __uint_as_float(0x7FFFFFFFu) : g.scale;
            }
        }
    }
}

// ------------------------------------------------------------ backward
//
// A block takes `tokens` tokens at a time and its groups their head rows; a lane keeps its columns, so that the weight's
// gradient is summed in registers over all of a block's rows, then over its groups in order, then over blocks by
// weight_sum.
struct HeadBackArgs {
    const float *dy, *x, *w, *rstd;
    float *dx, *part;
    Turn turn;
    int64_t rows, dy_s1, x_s1, dx_s1;
    int dim, heads, tokens;
};
constexpr int kBackTokens = 4, kBackRows = 2;

template <int LANES, int V, bool VEC>
__global__ void __launch_bounds__(kHeadThreads) heads_backward(HeadBackArgs a) {
    __shared__ __align__(16) float cs[kBackTokens][kMaxPairs], sn[kBackTokens][kMaxPairs];
    constexpr int GROUPS = kHeadWarps * 32 / LANES;
    __shared__ __align__(16) float sums[GROUPS][4 * V * LANES];
    const int l = threadIdx.x & (LANES - 1), group = threadIdx.x / LANES;
    const int pairs = a.turn.rot / 2;
    pdl_begin();
    float w[4 * V], acc[4 * V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int d = 4 * (l + LANES * v);
        float4 t = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (a.w && d < a.dim) t = load4<VEC>(a.w + d);
        w[4 * v] = t.x, w[4 * v + 1] = t.y, w[4 * v + 2] = t.z, w[4 * v + 3] = t.w;
    }
#pragma unroll
    for (int i = 0; i < 4 * V; ++i) acc[i] = 0.0f;
    for (int64_t first = (int64_t)blockIdx.x * a.tokens; first < a.rows; first += (int64_t)gridDim.x * a.tokens) {
        const int n = (int)min((int64_t)a.tokens, a.rows - first);
        if (pairs) {
            __syncthreads();
            for (int i = threadIdx.x; i < n * pairs; i += kHeadThreads) {
                const int tok = i / pairs, p = i - tok * pairs;
                const float2 t = turn_of(a.turn.pos[first + tok], a.turn.freq[p], a.turn.mag);
                cs[tok][p] = t.x, sn[tok][p] = t.y;
            }
            __syncthreads();
        }
        const int jobs = n * a.heads;
        for (int j0 = 0; j0 < jobs; j0 += GROUPS * kBackRows) {
            float u[kBackRows][4 * V], x[kBackRows][4 * V], rstd[kBackRows];
            int tok[kBackRows], head[kBackRows];
#pragma unroll
            for (int k = 0; k < kBackRows; ++k) {
                const int j = j0 + k * GROUPS + group;
                tok[k] = j < jobs ? j / a.heads : -1;
                head[k] = j - max(tok[k], 0) * a.heads;
                const int64_t row = first + max(tok[k], 0);
                rstd[k] = a.w && tok[k] >= 0 ? a.rstd[row * a.heads + head[k]] : 0.0f;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const int d = 4 * (l + LANES * v);
                    float4 t = make_float4(0.0f, 0.0f, 0.0f, 0.0f), z = t;
                    if (tok[k] >= 0 && d < a.dim) {
                        t = load4<VEC>(a.dy + row * a.dy_s1 + (int64_t)head[k] * a.dim + d);
                        if (a.w) z = load4<VEC>(a.x + row * a.x_s1 + (int64_t)head[k] * a.dim + d);
                    }
                    u[k][4 * v] = t.x, u[k][4 * v + 1] = t.y, u[k][4 * v + 2] = t.z, u[k][4 * v + 3] = t.w;
                    x[k][4 * v] = z.x, x[k][4 * v + 1] = z.y, x[k][4 * v + 2] = z.z, x[k][4 * v + 3] = z.w;
                }
            }
#pragma unroll
            for (int k = 0; k < kBackRows; ++k) {
                if (pairs) {
                    float c[4 * V] = {}, s[4 * V] = {};
                    turn_factors<LANES, V>(c, s, cs[max(tok[k], 0)], sn[max(tok[k], 0)], a.turn, l, true);
                    turn<LANES, V>(u[k], c, s, a.turn, l);
                }
                if (a.w) {
                    float dot = 0.0f;
#pragma unroll
                    for (int i = 0; i < 4 * V; ++i) {
                        acc[i] = fmaf(u[k][i], x[k][i] * rstd[k], acc[i]);
                        u[k][i] *= w[i];
                        dot = fmaf(u[k][i], x[k][i], dot);
                    }
                    const float m = group_sum<LANES>(dot) / (float)a.dim * (rstd[k] * rstd[k]);
#pragma unroll
                    for (int i = 0; i < 4 * V; ++i) u[k][i] = rstd[k] * fmaf(-x[k][i], m, u[k][i]);
                }
                if (tok[k] >= 0) {
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        const int d = 4 * (l + LANES * v);
                        if (d < a.dim)
                            store4<VEC>(a.dx + (first + tok[k]) * a.dx_s1 + (int64_t)head[k] * a.dim + d,
                                        make_float4(u[k][4 * v], u[k][4 * v + 1], u[k][4 * v + 2], u[k][4 * v + 3]));
                    }
                }
            }
        }
    }
    if (a.part) {
#pragma unroll
        for (int v = 0; v < V; ++v)
            *(float4*)&sums[group][4 * (l + LANES * v)] = make_float4(acc[4 * v], acc[4 * v + 1], acc[4 * v + 2], acc[4 * v + 3]);
        __syncthreads();
        for (int d = threadIdx.x; d < a.dim; d += kHeadThreads) {
            float t = 0.0f;
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) t += sums[g][d];
            a.part[(int64_t)blockIdx.x * a.dim + d] = t;
        }
    }
}

// dw[d] = sum of the blocks' parts, each of 32 warps an equal run of them.
__global__ void __launch_bounds__(1024) heads_weight_sum(float* dw, const float* part, int parts, int dim) {
    __shared__ float sh[32][33];
    pdl_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = blockIdx.x * 32 + lane, per = (parts + 31) / 32;
    float t = 0.0f;
    if (d < dim) {
#pragma unroll 8
        for (int p = warp * per; p < min(warp * per + per, parts); ++p) t += part[(int64_t)p * dim + d];
    }
    sh[warp][lane] = t;
    __syncthreads();
    t = warp_sum_f(sh[lane][warp]);
    if (lane == 0 && blockIdx.x * 32 + warp < dim) dw[blockIdx.x * 32 + warp] = t;
}

// ------------------------------------------------------------ cache read
//
// The rows' head rows of keys, then of values, in one order; a group takes every GROUPS-th of a run of kReadRows * GROUPS,
// all of its loads first.  Bound by HBM: 1 byte in and 4 out a value.
struct ReadArgs {
    const uint8_t *kq, *vq;
    const float *ks, *vs;
    float *k, *v;
    const int32_t* slot;
    int64_t rows, k_s1, v_s1;
    int dim, heads, page_log, slots;
};
constexpr int kReadRows = 4;

__device__ __forceinline__ float4 e4m3_values(uint32_t b) {
    uint32_t lo, hi;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"((uint16_t)b));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"((uint16_t)(b >> 16)));
    float4 r;
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}" : "=f"(r.x), "=f"(r.y) : "r"(lo));
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}" : "=f"(r.z), "=f"(r.w) : "r"(hi));
    return r;
}

template <int LANES, bool VEC>
__global__ void __launch_bounds__(kHeadThreads) cache_read(ReadArgs a) {
    constexpr int GROUPS = kHeadWarps * 32 / LANES;
    const int l = threadIdx.x & (LANES - 1), group = threadIdx.x / LANES;
    const int jobs = a.heads * ((a.k != nullptr) + (a.v != nullptr));
    const int64_t first = (int64_t)blockIdx.x * (GROUPS * kReadRows), row0 = first / jobs;
    const int rem = (int)(first - row0 * jobs);
    pdl_begin();
    uint32_t b[kReadRows];
    float s[kReadRows];
    float* to[kReadRows];
#pragma unroll
    for (int u = 0; u < kReadRows; ++u) {
        const int t = rem + u * GROUPS + group, up = t / jobs, j = t - up * jobs;
        const int64_t row = row0 + up;
        b[u] = 0, s[u] = 0.0f, to[u] = nullptr;
        if (row < a.rows && 4 * l < a.dim) {
            const bool value = !a.k || j >= a.heads;
            const int h = j - (a.k && value ? a.heads : 0), slot = a.slot[row];
            to[u] = (value ? a.v + row * a.v_s1 : a.k + row * a.k_s1) + (int64_t)h * a.dim + 4 * l;
            if ((uint32_t)slot < (uint32_t)a.slots) {
                const int64_t at = ((((int64_t)(slot >> a.page_log) * a.heads) + h) << a.page_log) + (slot & ((1 << a.page_log) - 1));
                b[u] = *(const uint32_t*)((value ? a.vq : a.kq) + at * a.dim + 4 * l);
                s[u] = (value ? a.vs : a.ks)[at];
            }
        }
    }
#pragma unroll
    for (int u = 0; u < kReadRows; ++u) {
        const float4 v = e4m3_values(b[u]);
        if (to[u]) store4<VEC>(to[u], make_float4(v.x * s[u], v.y * s[u], v.z * s[u], v.w * s[u]));
    }
}

constexpr int kSms = 148;

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
int log2_of(int v) {
    int n = 0;
    while ((1 << n) < v) ++n;
    return n;
}
Turn turn_args(const mag_cuda_rotation* r) { return Turn{r->pos, r->inv_freq, r->rot, r->interleaved != 0, r->magnitude}; }

template <int LANES, int V, bool VEC>
int run_forward(const HeadArgs& a, int64_t rows, cudaStream_t st) {
    constexpr int groups = kHeadWarps * 32 / LANES;
    const int jobs = a.q_heads + 2 * a.heads, few = (jobs + groups - 1) / groups, many = (jobs + 4 * groups - 1) / (4 * groups);
    // few tokens: a head row a group, so that more SMs share a token
    if (rows * many < kSms) return (int)launch_dep(heads_forward<LANES, V, 1, VEC>, dim3((unsigned)rows, (unsigned)few), dim3(kHeadThreads), 0, st, a);
    return (int)launch_dep(heads_forward<LANES, V, 4, VEC>, dim3((unsigned)rows, (unsigned)many), dim3(kHeadThreads), 0, st, a);
}
template <bool VEC>
int forward(const HeadArgs& a, int64_t rows, cudaStream_t st) {
    if (a.dim <= 64) return run_forward<16, 1, VEC>(a, rows, st);
    if (a.dim <= 128) return run_forward<32, 1, VEC>(a, rows, st);
    return run_forward<32, 2, VEC>(a, rows, st);
}

constexpr int kBackBlocks = 3 * kSms;
int back_tokens(int64_t rows) { return rows <= kBackBlocks ? 1 : kBackTokens; }
int back_blocks(int64_t rows) {
    const int64_t n = (rows + back_tokens(rows) - 1) / back_tokens(rows);
    return (int)(n < kBackBlocks ? n : kBackBlocks);
}
template <bool VEC>
int backward(const HeadBackArgs& a, cudaStream_t st) {
    const dim3 grid((unsigned)back_blocks(a.rows)), block(kHeadThreads);
    if (a.dim <= 64) return (int)launch_dep(heads_backward<16, 1, VEC>, grid, block, 0, st, a);
    if (a.dim <= 128) return (int)launch_dep(heads_backward<32, 1, VEC>, grid, block, 0, st, a);
    return (int)launch_dep(heads_backward<32, 2, VEC>, grid, block, 0, st, a);
}

template <bool VEC>
int read(const ReadArgs& a, cudaStream_t st) {
    const int64_t all = a.rows * a.heads * ((a.k != nullptr) + (a.v != nullptr)), per = kReadRows * (a.dim <= 64 ? 16 : 8);
    const dim3 grid((unsigned)((all + per - 1) / per)), block(kHeadThreads);
    if (a.dim <= 64) return (int)launch_dep(cache_read<16, VEC>, grid, block, 0, st, a);
    return (int)launch_dep(cache_read<32, VEC>, grid, block, 0, st, a);
}

}  // namespace

extern "C" int mcu_launch_rotate_heads(float* y, float* rstd, const float* x, const float* w, float eps, const mag_cuda_rotation* rot,
                                       int64_t rows, int64_t heads, int64_t head_dim, int64_t x_s1, int64_t y_s1, cudaStream_t st,
                                       int* launches) {
    HeadArgs a = {};
    a.q = x, a.q_w = w, a.q_out = y, a.rstd = rstd, a.turn = turn_args(rot), a.eps = eps;
    a.dim = (int)head_dim, a.q_heads = (int)heads, a.q_s1 = x_s1, a.out_s1 = y_s1;
    *launches = 1;
    const bool vec = aligned16(x) && aligned16(y) && aligned16(w) && !((x_s1 | y_s1) & 3);
    return vec ? forward<true>(a, rows, st) : forward<false>(a, rows, st);
}

extern "C" int mcu_launch_kv_write(const mag_cuda_kv_cache* cache, const int32_t* slot, const float* k, const float* v, const float* k_w,
                                   float* q_out, const float* q, const float* q_w, float eps, const mag_cuda_rotation* rot, int64_t rows,
                                   int64_t q_heads, int64_t k_s1, int64_t v_s1, int64_t q_s1, int64_t q_out_s1, cudaStream_t st,
                                   int* launches) {
    HeadArgs a = {};
    a.q = q, a.k = k, a.v = v, a.q_w = q_w, a.k_w = k_w, a.q_out = q_out;
    a.kq = cache->k, a.vq = cache->v, a.ks = cache->k_scale, a.vs = cache->v_scale, a.slot = slot;
    a.turn = turn_args(rot), a.eps = eps, a.dim = cache->head_dim, a.q_heads = (int)q_heads, a.heads = cache->heads;
    a.page_log = log2_of(cache->page_size), a.slots = cache->pages * cache->page_size;
    a.q_s1 = q_s1, a.k_s1 = k_s1, a.v_s1 = v_s1, a.out_s1 = q_out_s1;
    *launches = 1;
    const bool vec = aligned16(k) && aligned16(v) && aligned16(k_w) && aligned16(q) && aligned16(q_out) && aligned16(q_w) &&
                     !((k_s1 | v_s1) & 3) && (!q || !((q_s1 | q_out_s1) & 3));
    return vec ? forward<true>(a, rows, st) : forward<false>(a, rows, st);
}

extern "C" size_t mcu_rotate_heads_backward_scratch_bytes(int64_t rows, int64_t heads, int64_t head_dim) {
    (void)heads;
    return (size_t)back_blocks(rows) * (size_t)head_dim * 4;
}

extern "C" int mcu_launch_rotate_heads_backward(float* dx, float* dw, const float* dy, const float* x, const float* w, const float* rstd,
                                                const mag_cuda_rotation* rot, int64_t rows, int64_t heads, int64_t head_dim,
                                                int64_t dx_s1, int64_t dy_s1, int64_t x_s1, void* scratch, cudaStream_t st,
                                                int* launches) {
    const HeadBackArgs a{dy, x, w, rstd, dx, dw ? (float*)scratch : nullptr, turn_args(rot), rows, dy_s1, x_s1, dx_s1,
                         (int)head_dim, (int)heads, back_tokens(rows)};
    *launches = 1;
    const bool vec = aligned16(dx) && aligned16(dy) && aligned16(x) && aligned16(w) && !((dx_s1 | dy_s1) & 3) && (!x || !(x_s1 & 3));
    int rc = vec ? backward<true>(a, st) : backward<false>(a, st);
    if (!rc && dw) {
        rc = (int)launch_dep(heads_weight_sum, dim3((unsigned)((head_dim + 31) / 32)), dim3(1024), 0, st, dw, (const float*)scratch,
                             back_blocks(rows), (int)head_dim);
        ++*launches;
    }
    return rc;
}

extern "C" int mcu_launch_kv_read(const mag_cuda_kv_cache* cache, float* k, float* v, const int32_t* slot, int64_t rows, int64_t k_s1,
                                  int64_t v_s1, cudaStream_t st, int* launches) {
    const ReadArgs a{cache->k, cache->v, cache->k_scale, cache->v_scale, k, v, slot, rows, k_s1, v_s1, cache->head_dim, cache->heads,
                     log2_of(cache->page_size), cache->pages * cache->page_size};
    *launches = 1;
    const bool vec = aligned16(k) && aligned16(v) && (!k || !(k_s1 & 3)) && (!v || !(v_s1 & 3));
    return vec ? read<true>(a, st) : read<false>(a, st);
}
