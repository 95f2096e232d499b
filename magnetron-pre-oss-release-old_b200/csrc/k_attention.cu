// k_attention.cu - attention of new tokens over the paged e4m3 cache (mag_cuda_attention_paged_f32).
#include <cuda_runtime.h>
#include <cstdint>
#include "mcu_kernels.h"
#include "mcu_launch.cuh"
#include "mcu_lm.cuh"

using namespace mcu;

namespace {

__device__ __forceinline__ float4 e4m3_values(uint32_t b) {
    uint32_t lo, hi;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"((uint16_t)b));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"((uint16_t)(b >> 16)));
    float4 r;
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}" : "=f"(r.x), "=f"(r.y) : "r"(lo));
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}" : "=f"(r.z), "=f"(r.w) : "r"(hi));
    return r;
}

// A warp takes one head of one row and goes through its keys with the running maximum and sum.
__global__ void __launch_bounds__(128) attention_rows(mcu_attention a) {
    pdl_begin();
    const int lane = threadIdx.x & 31;
    const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5), row = item / a.q_heads;
    const int head = (int)(item - row * a.q_heads), dim = a.cache.head_dim, page = a.cache.page_size;
    if (row >= a.rows) return;
    int64_t seq = 0, s0 = 0, s1 = 0;
    for (; seq < a.seqs; ++seq) {
        s0 = min(max((int64_t)a.start[seq], (int64_t)0), a.rows);
        s1 = min(max((int64_t)a.start[seq + 1], s0), a.rows);
        if (row >= s0 && row < s1) break;
    }
    if (seq == a.seqs || row - s0 >= a.max_new) return;
    const int64_t length = min(max((int64_t)a.length[seq], (int64_t)0), a.table_s1 * page);
    const int64_t pos = length - (s1 - s0) + (row - s0), lo = a.window ? max(pos - a.window + 1, (int64_t)0) : 0;
    const int kv = head / (int)(a.q_heads / a.cache.heads);
    float4 q = make_float4(0.0f, 0.0f, 0.0f, 0.0f), o = q;
    if (4 * lane < dim) {
        const float* p = a.q + row * a.q_s1 + (int64_t)head * dim + 4 * lane;
        q = make_float4(p[0], p[1], p[2], p[3]);
    }
    float m = -INFINITY, l = 0.0f;
    for (int64_t j = lo; j <= pos; ++j) {
        const int pg = a.table[seq * a.table_s1 + j / page];
        if ((uint32_t)pg >= (uint32_t)a.cache.pages) continue;
        const int64_t at = ((int64_t)pg * a.cache.heads + kv) * page + j % page;
        float4 k = make_float4(0.0f, 0.0f, 0.0f, 0.0f), v = k;
        if (4 * lane < dim) {
            k = e4m3_values(*(const uint32_t*)(a.cache.k + at * dim + 4 * lane));
            v = e4m3_values(*(const uint32_t*)(a.cache.v + at * dim + 4 * lane));
        }
        const float vs = a.cache.v_scale[at];
        const float x = warp_sum_f(fmaf(q.x, k.x, fmaf(q.y, k.y, fmaf(q.z, k.z, q.w * k.w)))) * a.cache.k_scale[at] * a.scale;
        const float mn = fmaxf(m, x), f = m == mn ? 1.0f : expf(m - mn), p = x == -INFINITY ? 0.0f : expf(x - mn);
        l = fmaf(l, f, p);
        o.x = fmaf(o.x, f, p * (v.x * vs)), o.y = fmaf(o.y, f, p * (v.y * vs));
        o.z = fmaf(o.z, f, p * (v.z * vs)), o.w = fmaf(o.w, f, p * (v.w * vs));
        m = mn;
    }
    const float r = l == 0.0f ? 0.0f : 1.0f / l;
    if (4 * lane < dim) {
        float* p = a.out + row * a.out_s1 + (int64_t)head * dim + 4 * lane;
        p[0] = o.x * r, p[1] = o.y * r, p[2] = o.z * r, p[3] = o.w * r;
    }
    if (a.lse && lane == 0) a.lse[row * a.q_heads + head] = l == 0.0f ? -INFINITY : m + logf(l);
}

}  // namespace

extern "C" size_t mcu_attention_scratch_bytes(const mcu_attention* a) {
    (void)a;
    return 0;
}

extern "C" int mcu_launch_attention(const mcu_attention* a, void* scratch, int* status, cudaStream_t st, int* launches) {
    (void)scratch, (void)status;
    *launches = 1;
    return (int)launch_dep(attention_rows, dim3((unsigned)((a->rows * a->q_heads + 3) / 4)), dim3(128), 0, st, *a);
}
