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
constexpr int kMaxPairs = 128;  // of a token

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

// (cos, sin) of pos * f, times mag.  The angle is the product in f64 (31 and 24 bits, rounded to 53), reduced there to n quarter
// turns and |r| <= pi / 4 (pi / 2 as a sum of two f64); what r loses as an f32 is put back to first order, so that the results are
// within about an f32 rounding of that angle's.  The product's own rounding, at most 2^-53 of the angle, is half an f32 step of 1
// (2^-24) at most for angles below 2^30 and reaches 2^-23 at the last positions and a frequency of 1.
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

// A warp serves one token at a time.  It forms the token's cosines and sines in shared memory of its own (cs, then sn), and each
// lane keeps the factors of its values: y = x c + partner s.  All lanes take part.
template <int LANES, int V>
__device__ __forceinline__ void turn_factors(float (&c)[4 * V], float (&s)[4 * V], float* cs, const Turn& t, int64_t row, int l, bool back) {
    float* sn = cs + kMaxPairs;
    const int lane = threadIdx.x & 31, pos = t.pos[row];
    __syncwarp();  // (the last token's have been read)
    for (int i = lane; i < t.rot / 2; i += 32) {
        const float2 v = turn_of(pos, t.freq[i], t.mag);
        cs[i] = v.x, sn[i] = back ? -v.y : v.y;
    }
    __syncwarp();
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int d = 4 * (l + LANES * v);
        if (d >= t.rot) continue;
        if (t.pairs) {
            const float2 a = *(const float2*)(cs + d / 2), b = *(const float2*)(sn + d / 2);
            c[4 * v] = c[4 * v + 1] = a.x, c[4 * v + 2] = c[4 * v + 3] = a.y;
            s[4 * v] = -b.x, s[4 * v + 1] = b.x, s[4 * v + 2] = -b.y, s[4 * v + 3] = b.y;
        } else {
            const int half = t.rot / 2, p = d < half ? d : d - half;
            const float4 a = *(const float4*)(cs + p), b = *(const float4*)(sn + p);
            const float g = d < half ? -1.0f : 1.0f;
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

template <int LANES, int V, bool VEC>
__device__ __forceinline__ void load_row(float (&x)[4 * V], const float* p, int l, int dim) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int d = 4 * (l + LANES * v);
        float4 t = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (p && d < dim) t = load4<VEC>(p + d);
        x[4 * v] = t.x, x[4 * v + 1] = t.y, x[4 * v + 2] = t.z, x[4 * v + 3] = t.w;
    }
}
template <int LANES, int V, bool VEC>
__device__ __forceinline__ void store_row(float* p, const float (&x)[4 * V], int l, int dim) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int d = 4 * (l + LANES * v);
        if (d < dim) store4<VEC>(p + d, make_float4(x[4 * v], x[4 * v + 1], x[4 * v + 2], x[4 * v + 3]));
    }
}

// ------------------------------------------------------------ forward and cache write
//
// A warp takes a token and up to `rows_a_warp` of its head rows, U a group at a time.  Query rows go out in f32, key and value
// rows as e4m3 with their scale.
// What bounds it: instructions and HBM, one read and one write of each value.  The token's angles cost about two head rows' work, so
// that a warp serves 16 of them where there are enough warps; blocks that share a token's angles took longer (8191 x 32 x 128: 66 us
// with a token a block, of whose threads a quarter formed the angles; 82 with four tokens; 105 persistent; 51 so, 5.3 TB/s).  Rows
// of one kind run through one loop, whose addresses grow by constants: with the kind and the address of each row worked out row by
// row the same took 65 us, and a cache write of 8191 x (40 + 8 + 8) heads 100 instead of 83.
struct HeadArgs {
    const float *q, *k, *v, *q_w, *k_w;
    float *q_out, *rstd;
    uint8_t *kq, *vq;
    float *ks, *vs;
    const int32_t* slot;
    Turn turn;
    float eps, inv_dim;
    int dim, q_heads, heads, page_log, slots;  // heads: of keys and of values, 0 without a cache
    int rows_a_warp, shares;                   // head rows of a warp, and the warps that share a token
    int64_t rows, q_s1, k_s1, v_s1, out_s1;
};
constexpr int kForwardWarps = 4;

// What becomes of a run of `rows` head rows of one kind from `from` on, GROUPS at a time, U on their way.
enum Kind { QUERY, KEY, VALUE };
template <int LANES, int V, int U, bool VEC, int KIND>
__device__ __forceinline__ void head_run(const HeadArgs& a, const float* from, int rows, int64_t row, int first, const float* w, const float (&c)[4 * V],
                                         const float (&s)[4 * V], int64_t place) {
    constexpr int GROUPS = 32 / LANES;
    const int l = threadIdx.x & (LANES - 1), group = (threadIdx.x & 31) / LANES, step = GROUPS * a.dim;
    from += group * a.dim;
    float x[U][4 * V], f[4 * V];
#pragma unroll
    for (int u = 0; u < U; ++u) load_row<LANES, V, VEC>(x[u], u * GROUPS + group < rows ? from + u * step : nullptr, l, a.dim);
    if (KIND != VALUE && w) load_row<LANES, V, VEC>(f, w, l, a.dim);
    float* to = KIND == QUERY ? a.q_out + row * a.out_s1 + (int64_t)(first + group) * a.dim : nullptr;
    // (a head's rows of a page lie page_size rows apart)
    uint8_t* bytes = KIND == QUERY ? nullptr : (KIND == KEY ? a.kq : a.vq) + (place + ((int64_t)(first + group) << a.page_log)) * a.dim + 4 * l;
    float* scale = KIND == QUERY ? nullptr : (KIND == KEY ? a.ks : a.vs) + place + ((int64_t)(first + group) << a.page_log);
#pragma unroll 1
    for (int j = group; j < rows + group; j += U * GROUPS) {
        from += U * step;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool live = j + u * GROUPS < rows;
            float(&y)[4 * V] = x[u];
            if (KIND != VALUE && w) {
                float ss = 0.0f;
#pragma unroll
                for (int i = 0; i < 4 * V; ++i) ss = fmaf(y[i], y[i], ss);
                const float r = inv_sqrt(fmaf(group_sum<LANES>(ss), a.inv_dim, a.eps));
#pragma unroll
                for (int i = 0; i < 4 * V; ++i) y[i] = y[i] * r * f[i];
                if (KIND == QUERY && a.rstd && l == 0 && live) a.rstd[row * a.q_heads + first + j + u * GROUPS] = r;
            }
            if (KIND != VALUE && a.turn.rot) turn<LANES, V>(y, c, s, a.turn, l);
            if (KIND == QUERY) {
                if (live) store_row<LANES, V, VEC>(to + u * step, y, l, a.dim);
            } else if (V == 1) {  // (a cache's heads have at most 128 values)
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) top = max(top, abs_bits(y[i]));
                top = group_max<LANES>(top);
                if (live && place >= 0) {
                    const E4m3Group g = e4m3_group(top);
                    const bool bad = top >= 0x7F800000u;
                    const int64_t up = (int64_t)(u * GROUPS) << a.page_log;
                    if (4 * l < a.dim) *(uint32_t*)(bytes + up * a.dim) = bad ? 0u : e4m3_quotients(g, y[0], y[1], y[2], y[3]);
                    if (l == 0) scale[up] = bad ? __uint_as_float(0x7FFFFFFFu) : g.scale;
                }
            }
            load_row<LANES, V, VEC>(x[u], j + (u + U) * GROUPS < rows ? from + u * step : nullptr, l, a.dim);  // meanwhile
        }
        if (KIND == QUERY) {
            to += U * step;
        } else {
            const int64_t up = (int64_t)(U * GROUPS) << a.page_log;
            bytes += up * a.dim, scale += up;
        }
    }
}

template <int LANES, int V, int U, bool VEC, bool CACHE>
__global__ void __launch_bounds__(32 * kForwardWarps) heads_forward(HeadArgs a) {
    __shared__ __align__(16) float turns[kForwardWarps][2 * kMaxPairs];
    const int l = threadIdx.x & (LANES - 1), warp = threadIdx.x >> 5;
    const int64_t item = (int64_t)blockIdx.x * kForwardWarps + warp, row = item / a.shares;
    pdl_begin();
    if (row >= a.rows) return;
    const int j0 = (int)(item - row * a.shares) * a.rows_a_warp, j1 = min(j0 + a.rows_a_warp, a.q_heads + 2 * a.heads);
    float c[4 * V] = {}, s[4 * V] = {};
    if (a.turn.rot && j0 < a.q_heads + a.heads) turn_factors<LANES, V>(c, s, turns[warp], a.turn, row, l, false);
    if (j0 < a.q_heads)
        head_run<LANES, V, U, VEC, QUERY>(a, a.q + row * a.q_s1 + (int64_t)j0 * a.dim, min(j1, a.q_heads) - j0, row, j0, a.q_w, c, s, 0);
    if constexpr (CACHE) {
        const int slot = a.slot[row];
        const int64_t place =
            (uint32_t)slot < (uint32_t)a.slots ? (((int64_t)(slot >> a.page_log) * a.heads) << a.page_log) + (slot & ((1 << a.page_log) - 1)) : (int64_t)-1;
        const int k0 = max(j0 - a.q_heads, 0), k1 = min(j1 - a.q_heads, a.heads), v0 = max(j0 - a.q_heads - a.heads, 0), v1 = j1 - a.q_heads - a.heads;
        if (k0 < k1) head_run<LANES, V, U, VEC, KEY>(a, a.k + row * a.k_s1 + (int64_t)k0 * a.dim, k1 - k0, row, k0, a.k_w, c, s, place);
        if (v0 < v1) head_run<LANES, V, U, VEC, VALUE>(a, a.v + row * a.v_s1 + (int64_t)v0 * a.dim, v1 - v0, row, v0, nullptr, c, s, place);
    }
}

// ------------------------------------------------------------ backward
//
// Warps as in the forward pass, but they stay: a lane keeps its columns, so that the weight's gradient is summed in registers
// over all of a warp's rows, then over the block's groups in order, then over blocks by heads_weight_sum.  8191 x 32 x 128: 75 us,
// 5.4 TB/s of 12 bytes a value (102 with a block for a token).
struct HeadBackArgs {
    const float *dy, *x, *w, *rstd;
    float *dx, *part;
    Turn turn;
    int64_t rows, dy_s1, x_s1, dx_s1;
    float inv_dim;
    int dim, heads, rows_a_warp, shares;
};
constexpr int kBackRows = 2;

template <int LANES, int V, bool VEC>
__global__ void __launch_bounds__(kHeadThreads, V == 1 ? 4 : 2) heads_backward(HeadBackArgs a) {
    __shared__ __align__(16) float turns[kHeadWarps][2 * kMaxPairs];
    constexpr int GROUPS = 32 / LANES, ALL = kHeadWarps * GROUPS;
    __shared__ __align__(16) float sums[ALL][4 * V * LANES];
    const int l = threadIdx.x & (LANES - 1), group = (threadIdx.x & 31) / LANES, warp = threadIdx.x >> 5;
    pdl_begin();
    float w[4 * V], acc[4 * V];
    load_row<LANES, V, VEC>(w, a.w, l, a.dim);
#pragma unroll
    for (int i = 0; i < 4 * V; ++i) acc[i] = 0.0f;
    const int64_t items = a.rows * a.shares, all = (int64_t)gridDim.x * kHeadWarps;
#pragma unroll 1
    for (int64_t item = (int64_t)blockIdx.x * kHeadWarps + warp; item < items; item += all) {
        const int64_t row = item / a.shares;
        const int j0 = (int)(item - row * a.shares) * a.rows_a_warp, j1 = min(j0 + a.rows_a_warp, a.heads);
        const float *dy = a.dy + row * a.dy_s1, *xr = a.x + row * a.x_s1;
        float u[kBackRows][4 * V], x[kBackRows][4 * V], rstd[kBackRows], c[4 * V] = {}, s[4 * V] = {};
        auto load = [&](int k, int j) {
            const bool live = j < j1;
            rstd[k] = a.w && live ? a.rstd[row * a.heads + j] : 0.0f;
            load_row<LANES, V, VEC>(u[k], live ? dy + (int64_t)j * a.dim : nullptr, l, a.dim);
            load_row<LANES, V, VEC>(x[k], live && a.w ? xr + (int64_t)j * a.dim : nullptr, l, a.dim);
        };
#pragma unroll
        for (int k = 0; k < kBackRows; ++k) load(k, j0 + k * GROUPS + group);
        if (a.turn.rot) turn_factors<LANES, V>(c, s, turns[warp], a.turn, row, l, true);
#pragma unroll 1
        for (int jb = j0; jb < j1; jb += kBackRows * GROUPS) {
#pragma unroll
            for (int k = 0; k < kBackRows; ++k) {
                const int j = jb + k * GROUPS + group;
                if (a.turn.rot) turn<LANES, V>(u[k], c, s, a.turn, l);
                if (a.w) {
                    float dot = 0.0f;
#pragma unroll
                    for (int i = 0; i < 4 * V; ++i) {
                        acc[i] = fmaf(u[k][i], x[k][i] * rstd[k], acc[i]);
                        u[k][i] *= w[i];
                        dot = fmaf(u[k][i], x[k][i], dot);
                    }
                    const float m = group_sum<LANES>(dot) * a.inv_dim * (rstd[k] * rstd[k]);
#pragma unroll
                    for (int i = 0; i < 4 * V; ++i) u[k][i] = rstd[k] * fmaf(-x[k][i], m, u[k][i]);
                }
                if (j < j1) store_row<LANES, V, VEC>(a.dx + row * a.dx_s1 + (int64_t)j * a.dim, u[k], l, a.dim);
                load(k, j + kBackRows * GROUPS);
            }
        }
    }
    if (a.part) {
#pragma unroll
        for (int v = 0; v < V; ++v)
            *(float4*)&sums[warp * GROUPS + group][4 * (l + LANES * v)] = make_float4(acc[4 * v], acc[4 * v + 1], acc[4 * v + 2], acc[4 * v + 3]);
        __syncthreads();
        for (int d = threadIdx.x; d < a.dim; d += kHeadThreads) {
            float t = 0.0f;
#pragma unroll
            for (int g = 0; g < ALL; ++g) t += sums[g][d];
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
// A warp takes the keys or the values of a slot: its heads' rows lie page_size rows apart, so that one address serves them all;
// a lane holds four values, its group every GROUPS-th head, U on their way.  (Plain loads: the call before it may still write the cache when
// this kernel begins, so that its bytes are not read-only for it.)  Bound by HBM: 1 byte in and 4 out a value (with an
// address for every row it was bound by instructions, 137 us for 65000 x 8 x 128; 104 so, 6.4 TB/s).
struct ReadArgs {
    const uint8_t *kq, *vq;
    const float *ks, *vs;
    float *k, *v;
    const int32_t* slot;
    int64_t rows, k_s1, v_s1;
    int dim, heads, page_log, slots, shares, rows_a_warp;
};

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
    constexpr int GROUPS = 32 / LANES, U = 4;
    const int l = threadIdx.x & (LANES - 1), group = (threadIdx.x & 31) / LANES;
    const int both = (a.k != nullptr) + (a.v != nullptr);
    const int64_t item = (int64_t)blockIdx.x * kHeadWarps + (threadIdx.x >> 5), row = item / (both * a.shares);
    pdl_begin();
    if (row >= a.rows) return;
    const int part = (int)(item - row * (both * a.shares)), share = part >> (both - 1);
    const bool value = both == 2 ? part & 1 : a.v != nullptr;
    const int j0 = share * a.rows_a_warp + group, j1 = min(share * a.rows_a_warp + a.rows_a_warp, a.heads), slot = a.slot[row];
    const bool there = (uint32_t)slot < (uint32_t)a.slots;
    const int64_t place = there ? (((int64_t)(slot >> a.page_log) * a.heads + j0) << a.page_log) + (slot & ((1 << a.page_log) - 1)) : 0;
    const uint8_t* bytes = (value ? a.vq : a.kq) + place * a.dim + 4 * l;
    const float* scale = (value ? a.vs : a.ks) + place;
    float* to = (value ? a.v + row * a.v_s1 : a.k + row * a.k_s1) + (int64_t)j0 * a.dim + 4 * l;
    const int64_t up = (int64_t)GROUPS << a.page_log, up_bytes = up * a.dim;
    if (4 * l >= a.dim) return;
#pragma unroll 1
    for (int j = j0; j < j1; j += U * GROUPS) {
        uint32_t b[U];
        float s[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool live = there && j + u * GROUPS < j1;
            b[u] = live ? *(const uint32_t*)(bytes + u * up_bytes) : 0u;
            s[u] = live ? scale[u * up] : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float4 v = e4m3_values(b[u]);
            if (j + u * GROUPS < j1) store4<VEC>(to + u * GROUPS * a.dim, make_float4(v.x * s[u], v.y * s[u], v.z * s[u], v.w * s[u]));
        }
        bytes += U * up_bytes, scale += U * up, to += U * GROUPS * a.dim;
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

// Head rows of a warp: 16 of them share the token's angles where that leaves two warps a scheduler's slot, fewer for few tokens,
// down to one step of a warp (least).
int rows_a_warp(int64_t rows, int jobs, int least) {
    int n = 16;
    while (n > least && rows * ((jobs + n - 1) / n) < (int64_t)kSms * 64) n /= 2;
    return n;
}

template <int LANES, int V, bool VEC>
int run_forward(HeadArgs& a, int64_t rows, cudaStream_t st) {
    const int jobs = a.q_heads + 2 * a.heads;
    a.rows = rows, a.inv_dim = 1.0f / (float)a.dim;
    a.rows_a_warp = rows_a_warp(rows, jobs, 32 / LANES), a.shares = (jobs + a.rows_a_warp - 1) / a.rows_a_warp;
    const dim3 grid((unsigned)((rows * a.shares + kForwardWarps - 1) / kForwardWarps)), block(32 * kForwardWarps);
    constexpr int U = V == 1 ? 4 : 2;
    if constexpr (V == 1) {
        if (a.heads)
            return (int)(a.rows_a_warp < 4 ? launch_dep(heads_forward<LANES, V, 1, VEC, true>, grid, block, 0, st, a)
                                           : launch_dep(heads_forward<LANES, V, U, VEC, true>, grid, block, 0, st, a));
    }
    return (int)(a.rows_a_warp < 4 ? launch_dep(heads_forward<LANES, V, 1, VEC, false>, grid, block, 0, st, a)
                                   : launch_dep(heads_forward<LANES, V, U, VEC, false>, grid, block, 0, st, a));
}
template <bool VEC>
int forward(HeadArgs& a, int64_t rows, cudaStream_t st) {
    if (a.dim <= 64) return run_forward<16, 1, VEC>(a, rows, st);
    if (a.dim <= 128) return run_forward<32, 1, VEC>(a, rows, st);
    return run_forward<32, 2, VEC>(a, rows, st);
}

constexpr int kBackBlocks = 4 * kSms;
int back_share(int64_t rows, int64_t heads, int64_t dim) { return rows_a_warp(rows, (int)heads, dim <= 64 ? 4 : 2); }
int back_blocks(int64_t rows, int64_t heads, int64_t dim) {
    const int share = back_share(rows, heads, dim);
    const int64_t n = (rows * ((heads + share - 1) / share) + kHeadWarps - 1) / kHeadWarps;
    return (int)(n < kBackBlocks ? n : kBackBlocks);
}
template <bool VEC>
int backward(HeadBackArgs& a, cudaStream_t st) {
    a.rows_a_warp = back_share(a.rows, a.heads, a.dim), a.shares = (a.heads + a.rows_a_warp - 1) / a.rows_a_warp;
    const dim3 grid((unsigned)back_blocks(a.rows, a.heads, a.dim)), block(kHeadThreads);
    if (a.dim <= 64) return (int)launch_dep(heads_backward<16, 1, VEC>, grid, block, 0, st, a);
    if (a.dim <= 128) return (int)launch_dep(heads_backward<32, 1, VEC>, grid, block, 0, st, a);
    return (int)launch_dep(heads_backward<32, 2, VEC>, grid, block, 0, st, a);
}

template <bool VEC>
int read(ReadArgs& a, cudaStream_t st) {
    const int both = (a.k != nullptr) + (a.v != nullptr);
    a.rows_a_warp = rows_a_warp(a.rows * both, a.heads, a.dim <= 64 ? 2 : 1), a.shares = (a.heads + a.rows_a_warp - 1) / a.rows_a_warp;
    const dim3 grid((unsigned)((a.rows * both * a.shares + kHeadWarps - 1) / kHeadWarps)), block(kHeadThreads);
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
    return (size_t)back_blocks(rows, heads, head_dim) * (size_t)head_dim * 4;
}

extern "C" int mcu_launch_rotate_heads_backward(float* dx, float* dw, const float* dy, const float* x, const float* w, const float* rstd,
                                                const mag_cuda_rotation* rot, int64_t rows, int64_t heads, int64_t head_dim,
                                                int64_t dx_s1, int64_t dy_s1, int64_t x_s1, void* scratch, cudaStream_t st,
                                                int* launches) {
    HeadBackArgs a{dy, x, w, rstd, dx, dw ? (float*)scratch : nullptr, turn_args(rot), rows, dy_s1, x_s1, dx_s1,
                   1.0f / (float)head_dim, (int)head_dim, (int)heads, 0, 0};
    *launches = 1;
    const bool vec = aligned16(dx) && aligned16(dy) && aligned16(x) && aligned16(w) && !((dx_s1 | dy_s1) & 3) && (!x || !(x_s1 & 3));
    int rc = vec ? backward<true>(a, st) : backward<false>(a, st);
    if (!rc && dw) {
        rc = (int)launch_dep(heads_weight_sum, dim3((unsigned)((head_dim + 31) / 32)), dim3(1024), 0, st, dw, (const float*)scratch,
                             back_blocks(rows, heads, head_dim), (int)head_dim);
        ++*launches;
    }
    return rc;
}

extern "C" int mcu_launch_kv_read(const mag_cuda_kv_cache* cache, float* k, float* v, const int32_t* slot, int64_t rows, int64_t k_s1,
                                  int64_t v_s1, cudaStream_t st, int* launches) {
    ReadArgs a{cache->k, cache->v, cache->k_scale, cache->v_scale, k, v, slot, rows, k_s1, v_s1, cache->head_dim, cache->heads,
               log2_of(cache->page_size), cache->pages * cache->page_size, 0, 0};
    *launches = 1;
    const bool vec = aligned16(k) && aligned16(v) && (!k || !(k_s1 & 3)) && (!v || !(v_s1 & 3));
    return vec ? read<true>(a, st) : read<false>(a, st);
}
