// k_attention.cu - attention of new tokens over the paged e4m3 cache (mag_cuda_attention_paged_f32).
#include <cuda_runtime.h>
#include <cstdint>
#include "mcu_attention.cuh"
#include "mcu_attention_tiles.cuh"
#include "mcu_device.h"

using namespace mcu;

namespace {

// ------------------------------------------------------------ few rows: single tokens and short runs of them
//
// The rows of one kv head (new tokens x query heads of the group) are at most 16 here, so the cache's bytes bound the
// work: each is read once, by one warp, for all rows.  A block works through its share of all (sequence, kv head) items'
// units of 128 tokens; its warps take groups of 16 tokens in turn, two or three on their way by cp.async in a ring of the warp's
// own, and each keeps its own running maximum, sum and output, and for each row the unit of its weights (the largest probability times
// scale so far).  The block's warps are joined in shared memory when an item ends; of the blocks that share an item the last one joins
// their parts.
//
// Products run on mma.sync m16n8k16 (f16, f32 sums): e4m3 bytes become f16 in registers, exactly.  Queries and
// weights are split in two f16, high and low.  Up to 8 rows (STACK) the halves are rows 0-7 and 8-15 of one
// operand, so that the split costs no instruction and a thread finds both halves' results in its own registers.
// The order of a product's inner index is free, so it is chosen such that a thread's operands are 16 consecutive bytes
// of a row of keys (inner index: the head's values) and of four rows of values (columns: the head's values).
//
// Measured (32 query heads on 8 of 128): 64 sequences of up to 16000 tokens 271 us in runs of a second, 5.2 TB/s of the cache, when
// the power limit lowers the clock (234 in runs of some milliseconds); four of up to 2000
// tokens 13 us, which is latency: about 1.6 us to find the share, 1.3 to the first copies, 2.5 for the groups, 0.8 to join the warps,
// and three to four of fences, counter and the parts' join, at the pace of code that runs once.  (Short runs of one block of twelve
// warps an SM: the former took 306 us with eight warps of four stages, 264 with a second launch that joins the parts, 255 without.)  Up
// to 16 rows: 404 us with 128 query heads; with one unit of scales for a warp instead of one for a row 384, but rows lost bits beside
// others' large values.
constexpr int kSms = 148;
constexpr int kGroup = 16;               // tokens of a warp's step; pages hold a multiple
constexpr float kLowest = -3.402823466e38f;  // the maximum of no logits
constexpr int kFlush = 16;               // groups between two flushes: the tensor core's sums lose up to a step each

template <int DP, bool STACK, int BLOCKS>
struct FewCfg {
    static constexpr int WARPS = (STACK ? 12 : 8) / BLOCKS, STAGES = STACK ? 3 : 4;
    static constexpr int STAGE = 2 * kGroup * DP + 2 * kGroup * 4;  // keys, values, their scales
    static constexpr int RING = STAGES * STAGE;
};
template <int DP, bool STACK, int BLOCKS>
struct FewSmem {
    static constexpr int VALS = (STACK ? DP / 4 : DP / 2);  // outputs a thread holds
    static constexpr int WARPS = FewCfg<DP, STACK, BLOCKS>::WARPS;
    static constexpr int SUMS = FewCfg<DP, STACK, BLOCKS>::RING * WARPS;
    static constexpr int STATS = SUMS + WARPS * 32 * VALS * 4;  // [warp][16] of (m, l), then [warp][16] of the outputs' unit, 16 ints
    static constexpr int BYTES = STATS + WARPS * 16 * 12 + 64;
    static_assert(BLOCKS * (BYTES + 1024) <= 228 * 1024, "must fit shared memory");
    static_assert(Share<16, DP, 32 * WARPS>::SMEM <= SUMS, "the search for work takes the rings' room");
};

__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four values of an item's row from column d on, normed by the sum `total` of 2^(logit - top): to out, with the row's lse, where
// the block has the whole item, else to the block's slot.
template <int DP, int THREADS>
__device__ __forceinline__ void put_out(const AttnArgs& a, const Share<16, DP, THREADS>& sh, const Item& it, int row, int d, float4 v, float top,
                                        float total) {
    if (it.from == 0 && it.to == it.units) {
        const int r = it.first_row + row, token = r / a.group, head = it.head * a.group + r % a.group;
        store_row(a, it.row0 + token, head, d, v);
        if (d == 0 && a.lse) a.lse[(int64_t)(it.row0 + token) * a.heads * a.group + head] = total == 0.0f ? -INFINITY : (top + log2f(total)) * kLn2;
        return;
    }
    float* p = sh.slot(a, it.from == 0);
    if (d == 0) p[8 + 2 * row] = top, p[9 + 2 * row] = total;
    *(float4*)(p + 8 + 2 * 16 + row * DP + d) = v;
}

// EXACT: the head has DP values, so that a group's rows lie at constant distances.
template <int DP, bool STACK, bool EXACT, int BLOCKS>
__global__ void __launch_bounds__(32 * FewCfg<DP, STACK, BLOCKS>::WARPS, BLOCKS) attention_few(AttnArgs a) {
    using C = FewCfg<DP, STACK, BLOCKS>;
    constexpr int kFewWarps = C::WARPS, kFewStages = C::STAGES;
    using S = FewSmem<DP, STACK, BLOCKS>;
    extern __shared__ __align__(128) uint8_t smem[];
    constexpr int KI = DP / 64;      // 16-byte pieces of a key a thread holds
    constexpr int NT = DP / 8;       // column tiles of the output
    constexpr int VB = DP / 8;       // bytes of a row of values a thread holds
    constexpr int QF = STACK ? 1 : 2;
    constexpr int NR = STACK ? 1 : 2;  // rows a thread works on: g, and g + 8
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const uint32_t ring = smem_addr(smem) + warp * C::RING;
    float4* sums = (float4*)(smem + S::SUMS) + warp * 8 * S::VALS;  // [VALS / 4][32]
    float2* stats = (float2*)(smem + S::STATS);
    float* units = (float*)(stats + kFewWarps * 16);
    int* cut = (int*)(units + kFewWarps * 16);  // what an item that ends, or begins, elsewhere is: 8 ints each
    pdl_begin();

    Share<16, DP, 32 * kFewWarps> sh;
    if (threadIdx.x < 16) cut[threadIdx.x] = 0;
    if (!sh.find(a, (int64_t*)smem)) return;
    if (!EXACT) {  // columns past the head's stay zero: no copy writes them
        for (int i = lane; i < C::RING / 16; i += 32) *(uint4*)(smem + warp * C::RING + 16 * i) = make_uint4(0, 0, 0, 0);
        __syncwarp();
    }
    while (sh.more()) {
        const Item it = sh.item(a);
        const int rows = it.rows;
        // ---- what each row sees, and what all rows do
        int first[NR], last[NR];
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const int row = g + 8 * r;
            last[r] = row < rows ? it.pos + row / a.group : -1;
            first[r] = a.window && last[r] >= a.window ? last[r] - a.window + 1 : 0;
        }
        const int all_last = it.pos, all_first = it.top_first;  // tokens within are seen by every row

        float o[NT][4];
#pragma unroll
        for (int j = 0; j < NT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
        float m[NR], l[NR], fade[NR], per[NR];  // per: 1 / the unit of the row's weights
#pragma unroll
        for (int r = 0; r < NR; ++r) m[r] = kLowest, l[r] = 0.0f, fade[r] = 1.0f, per[r] = 1.0f / kLeastUnit;
#pragma unroll
        for (int e = 0; e < S::VALS / 4; ++e) sums[e * 32 + lane] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);

        const int g0 = it.from * 8 + warp, g1 = min(it.to * 8, (it.high - it.base + kGroup - 1) / kGroup);
        const int steps = g0 < g1 ? (g1 - g0 + kFewWarps - 1) / kFewWarps : 0;
        const int32_t* table = a.table + (int64_t)it.seq * a.table_s1;
        int page = steps > 0 ? table[(it.base + kGroup * g0) >> a.page_log] : -1;
        uint32_t there = 0;               // bit s: the group in stage s has a page
        int issued = 0, to = 0;           // groups issued, and the next one's stage
        int next = it.base + kGroup * g0;  // its first token
        auto issue = [&]() {
            if (issued < steps) {
                const bool ok = (uint32_t)page < (uint32_t)a.pages;
                there = (there & ~(1u << to)) | ((uint32_t)ok << to);
                if (ok) {
                    const int64_t at = ((((int64_t)page * a.heads) + it.head) << a.page_log) + (next & ((1 << a.page_log) - 1));
                    constexpr int PR = 512 / DP;  // rows of one copy of the warp
                    const int r0 = lane / (DP / 16), ch = lane % (DP / 16), dim = EXACT ? DP : a.dim;
                    const int64_t from = (at + r0) * dim + 16 * ch;
                    const uint8_t *pk = a.k + from, *pv = a.v + from;
                    const uint32_t dst = ring + to * C::STAGE + r0 * DP;
                    // (row r0 + PR i has r0's place among the swizzled pieces, but for values of 128 that of two)
                    const uint32_t kd = dst + 16 * key_chunk<DP>(ch, r0), vd = dst + kGroup * DP + 16 * value_chunk<DP>(ch, r0);
                    if (EXACT && next >= it.low && next + kGroup <= it.high) {
#pragma unroll
                        for (int i = 0; i < kGroup / PR; ++i) {
                            copy16(kd + i * PR * DP, pk + i * PR * DP);
                            copy16((vd ^ value_turn<DP>(i)) + i * PR * DP, pv + i * PR * DP);
                        }
                    } else if (EXACT || 16 * ch < dim) {
#pragma unroll
                        for (int i = 0; i < kGroup / PR; ++i) {
                            const int j = next + r0 + PR * i;
                            const bool in = j >= it.low && j < it.high;
                            copy16(kd + i * PR * DP, pk + i * PR * dim, in);
                            copy16((vd ^ value_turn<DP>(i)) + i * PR * DP, pv + i * PR * dim, in);
                        }
                    }
                    if (lane < 8) copy16(ring + to * C::STAGE + 2 * kGroup * DP + 16 * lane, (lane < 4 ? a.ks : a.vs) + at + 4 * (lane & 3));
                }
                next += kFewWarps * kGroup;
                if (issued + 1 < steps) page = table[next >> a.page_log];
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            ++issued, to = to == kFewStages - 1 ? 0 : to + 1;
        };
        auto flush = [&]() {
#pragma unroll
            for (int r = 0; r < NR; ++r)
#pragma unroll
                for (int e = 0; e < DP / 16; ++e) {  // half of the columns, four tiles
                    float4 t = sums[(r * (DP / 16) + e) * 32 + lane];
                    const int half = e / (DP / 32), j = 4 * (e % (DP / 32));
                    float v[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[k] = STACK ? o[j + k][half] + o[j + k][2 + half] : o[j + k][2 * r + half];
                    t.x = fmaf(t.x, fade[r], v[0]), t.y = fmaf(t.y, fade[r], v[1]), t.z = fmaf(t.z, fade[r], v[2]), t.w = fmaf(t.w, fade[r], v[3]);
                    sums[(r * (DP / 16) + e) * 32 + lane] = t;
                }
#pragma unroll
            for (int j = 0; j < NT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
#pragma unroll
            for (int r = 0; r < NR; ++r) fade[r] = 1.0f;
        };
#pragma unroll
        for (int s = 0; s < kFewStages - 1; ++s) issue();
        // ---- queries: operand fragments and each row's factor to log2 units
        uint32_t qf[QF][4 * KI][4];
        float rf[NR];
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const int row = g + 8 * r;
            float x[KI][16];
            uint32_t top = 0;
            const bool live = row < rows;
            const float* p = a.q + (int64_t)(it.row0 + (live ? row / a.group : 0)) * a.q_s1 +
                             (int64_t)(it.head * a.group + (live ? row % a.group : 0)) * a.dim;
#pragma unroll
            for (int i = 0; i < KI; ++i) {
                const int d = 64 * i + 16 * c;
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const float4 t = live && d < a.dim ? four_of(p + d + 4 * v, a.q_vec) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    x[i][4 * v] = t.x, x[i][4 * v + 1] = t.y, x[i][4 * v + 2] = t.z, x[i][4 * v + 3] = t.w;
                }
#pragma unroll
                for (int v = 0; v < 16; ++v) top = max(top, abs_bits(x[i][v]));
            }
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float up = query_unit(top);
            rf[r] = logit_unit(a.scale, up);
#pragma unroll
            for (int i = 0; i < KI; ++i)
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    uint32_t h0, l0, h1, l1;
                    split2(x[i][4 * s] * up, x[i][4 * s + 1] * up, h0, l0);
                    split2(x[i][4 * s + 2] * up, x[i][4 * s + 3] * up, h1, l1);
                    if (STACK) {
                        qf[0][4 * i + s][0] = h0, qf[0][4 * i + s][1] = l0, qf[0][4 * i + s][2] = h1, qf[0][4 * i + s][3] = l1;
                    } else {
                        qf[0][4 * i + s][r] = h0, qf[0][4 * i + s][2 + r] = h1;
                        qf[QF - 1][4 * i + s][r] = l0, qf[QF - 1][4 * i + s][2 + r] = l1;
                    }
                }
        }
        int first_token = it.base + kGroup * g0;
        const int key0 = g * DP + 16 * key_chunk<DP>(c, g), value0 = kGroup * DP + 2 * c * DP + 16 * value_chunk<DP>(DP == 128 ? g : g >> 1, 2 * c) + (DP == 128 ? 0 : 8 * (g & 1));
        for (int i = 0, st = kFewStages - 1, summed = 0; i < steps; ++i) {  // summed: groups since the last flush
            asm volatile("cp.async.wait_group %0;" ::"n"(kFewStages - 2) : "memory");
            __syncwarp();
            st = st == kFewStages - 1 ? 0 : st + 1;
            const int j0 = first_token;
            first_token += kFewWarps * kGroup;
            const bool has = there >> st & 1;
            issue();
            if (!has) continue;  // (the same for the whole warp)
            const uint8_t* at = smem + warp * C::RING + st * C::STAGE;
            // ---- logits of 16 tokens: tiles of 8, the inner index in the order of the thread's bytes
            float s[2][4];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.0f;
#pragma unroll
                for (int p = 0; p < KI; ++p) {
                    const uint4 w = *(const uint4*)(at + 8 * t * DP + (key0 ^ 64 * p));  // (piece 4 p + c of row 8 t + g)
                    const uint32_t b[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t b0 = f16_of_e4m3(b[k]), b1 = f16_of_e4m3(b[k] >> 16);
#pragma unroll
                        for (int f = 0; f < QF; ++f) mma16(s[t], qf[f][4 * p + k], b0, b1);
                    }
                }
            }
            float ks[4], vs[4];
            {
                const float2* f = (const float2*)(at + 2 * kGroup * DP) + c;
                const float2 k0 = f[0], k1 = f[4], v0 = f[8], v1 = f[12];
                ks[0] = k0.x, ks[1] = k0.y, ks[2] = k1.x, ks[3] = k1.y, vs[0] = v0.x, vs[1] = v0.y, vs[2] = v1.x, vs[3] = v1.y;
            }
            const bool edge = j0 < all_first || j0 + kGroup - 1 > all_last;
            float t[NR][4];
            bool seen[NR][4];
#pragma unroll
            for (int r = 0; r < NR; ++r)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float raw = STACK ? s[k >> 1][k & 1] + s[k >> 1][2 + (k & 1)] : s[k >> 1][2 * r + (k & 1)];
                    t[r][k] = __fmul_rn(raw, ks[k]);
                    seen[r][k] = true;
                }
            if (edge) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int j = j0 + 8 * (k >> 1) + 2 * c + (k & 1);
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        seen[r][k] = j >= first[r] && j <= last[r];
                        if (!seen[r][k]) t[r][k] = -INFINITY;
                    }
                }
            }
            // ---- probabilities and weights (probability times the value's scale, in the row's unit); the running maxima and the
            // units, where one of them grows
            float p[NR][4], w[NR][4];
            auto weigh = [&]() {
#pragma unroll
                for (int r = 0; r < NR; ++r)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float e = exp2_f(fmaf(t[r][k] - m[r], rf[r], kTop));
                        p[r][k] = e;  // (zero for -inf)
                        w[r][k] = seen[r][k] ? e * per[r] * vs[k] : 0.0f;  // (in this order: neither product overflows)
                    }
            };
            weigh();
            bool grows = false;
#pragma unroll
            for (int r = 0; r < NR; ++r)
                grows |= fmaxf(fmaxf(t[r][0], t[r][1]), fmaxf(t[r][2], t[r][3])) > m[r] || fmaxf(fmaxf(w[r][0], w[r][1]), fmaxf(w[r][2], w[r][3])) > 0x1p15f;
            if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    float x = fmaxf(fmaxf(t[r][0], t[r][1]), fmaxf(t[r][2], t[r][3]));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
                    float f = 1.0f;
                    if (x > m[r]) {
                        f = exp2_f((m[r] - x) * rf[r]);
                        m[r] = x;
                        l[r] *= f;
                    }
                    float big = 0.0f;  // the largest weight, as it is
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (seen[r][k]) big = fmaxf(big, exp2_f((t[r][k] - m[r]) * rf[r]) * vs[k]);
                    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
                    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
                    const float held = one_by(per[r]) * f;  // what the older weights' unit has become
                    const float unit = fmaxf(unit_from(fmaxf(held, kLeastUnit)), big > kLeastUnit && big < kLargestScale ? unit_above(big) : 0.0f);
                    per[r] = one_by(unit);
                    f = held * per[r];
                    fade[r] *= f;
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        o[j][2 * r] *= f, o[j][2 * r + 1] *= f;
                        if (STACK) o[j][2] *= f, o[j][3] *= f;
                    }
                }
                weigh();
            }
            // ---- as operand fragments
            uint32_t pf[QF][4];
#pragma unroll
            for (int r = 0; r < NR; ++r) {
#pragma unroll
                for (int k = 0; k < 4; ++k) l[r] += p[r][k];
                uint32_t h0, l0, h1, l1;
                split2(w[r][0], w[r][1], h0, l0);
                split2(w[r][2], w[r][3], h1, l1);
                if (STACK) {
                    pf[0][0] = h0, pf[0][1] = l0, pf[0][2] = h1, pf[0][3] = l1;
                } else {
                    pf[0][r] = h0, pf[0][2 + r] = h1;
                    pf[QF - 1][r] = l0, pf[QF - 1][2 + r] = l1;
                }
            }
            // ---- output: 16 tokens are the inner index, a thread holds VB bytes of the four rows of its tokens
            uint32_t b[4][VB / 4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint8_t* va = at + value0 + (8 * (k >> 1) + (k & 1)) * DP;  // row 8 (k / 2) + 2 c + k % 2
                if (DP == 128) {
                    const uint4 w = *(const uint4*)va;
                    b[k][0] = w.x, b[k][1] = w.y, b[k][VB / 4 - 2] = w.z, b[k][VB / 4 - 1] = w.w;
                } else {
                    const uint2 w = *(const uint2*)va;
                    b[k][0] = w.x, b[k][1] = w.y;
                }
            }
#pragma unroll
            for (int w = 0; w < VB / 4; ++w)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t x = __byte_perm(b[0][w], b[1][w], h ? 0x7362 : 0x5140), y = __byte_perm(b[2][w], b[3][w], h ? 0x7362 : 0x5140);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const uint32_t b0 = f16_of_e4m3(k ? x >> 16 : x), b1 = f16_of_e4m3(k ? y >> 16 : y);
#pragma unroll
                        for (int f = 0; f < QF; ++f) mma16(o[4 * w + 2 * h + k], pf[f], b0, b1);
                    }
                }
            if (++summed == kFlush) flush(), summed = 0;
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        flush();
        // ---- the block's warps joined
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            if (c == 0) stats[warp * 16 + g + 8 * r] = make_float2(m[r] == kLowest ? kNone : top_of(m[r], rf[r]), l[r]), units[warp * 16 + g + 8 * r] = one_by(per[r]);
        }
        const bool whole = it.from == 0 && it.to == it.units;
        if (!whole && warp == kFewWarps - 1 && lane == 0) {
            int* c = cut + 8 * (it.from == 0);
            c[0] = sh.first_block(it), c[1] = sh.last_block(it) - c[0] + 1, c[2] = rows, c[3] = it.row0, c[4] = it.head * a.group;
        }
        __syncthreads();
        for (int x = threadIdx.x; x < 8 * S::VALS; x += 32 * kFewWarps) {
            const int e = x >> 5, ln = x & 31, r = e / (DP / 16), row = (ln >> 2) + 8 * r;
            const int half = e % (DP / 16) / (DP / 32), j = 4 * (e % (DP / 32)), d = VB * (2 * (ln & 3) + half) + j;
            if (row >= rows || d >= a.dim) continue;
            float top = kNone, total = 0.0f;
#pragma unroll
            for (int w = 0; w < kFewWarps; ++w) top = fmaxf(top, stats[w * 16 + row].x);
            float f[kFewWarps];
#pragma unroll
            for (int w = 0; w < kFewWarps; ++w) {
                const float2 st = stats[w * 16 + row];
                f[w] = exp2_f(st.x - top);
                total = fmaf(st.y, f[w], total);
            }
            const float inv = total == 0.0f ? 0.0f : 1.0f / total;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kFewWarps; ++w) {
                const float4 t = ((float4*)(smem + S::SUMS))[w * 8 * S::VALS + x];
                const float k = f[w] * inv, unit = units[w * 16 + row];  // (their product may be less than f32 holds)
                v.x = fmaf(t.x * k, unit, v.x), v.y = fmaf(t.y * k, unit, v.y), v.z = fmaf(t.z * k, unit, v.z), v.w = fmaf(t.w * k, unit, v.w);
            }
            put_out(a, sh, it, row, d, v, top, total);
        }
        __syncthreads();
        sh.advance(a, it);
    }
    // ---- items that other blocks have parts of, one at either end of the block's share at most: the last of an item's blocks
    // joins its parts.  The item's counter returns to zero with it.
    __threadfence();
    __syncthreads();
    if (threadIdx.x < 2) {
        int* c = cut + 8 * threadIdx.x;
        c[5] = c[1] && atomicInc(a.joins + c[0], (uint32_t)(c[1] - 1)) == (uint32_t)(c[1] - 1);
    }
    __syncthreads();
    for (int w = 0; w < 2; ++w) {
        const int* c = cut + 8 * w;
        if (!c[5]) continue;
        __threadfence();
        for (int r = warp; r < c[2]; r += kFewWarps) join_row<16, DP>(a, c[0], c[1], r, c[3] + r / a.group, c[4] + r % a.group);
    }
}

template <int DP, bool STACK, bool EXACT, int BLOCKS>
int run_few(const AttnArgs& a, cudaStream_t st) {
    static bool done[64];
    constexpr int bytes = FewSmem<DP, STACK, BLOCKS>::BYTES;
    const cudaError_t e = allow_smem(attention_few<DP, STACK, EXACT, BLOCKS>, bytes, done);
    if (e != cudaSuccess) return (int)e;
    return (int)launch_dep(attention_few<DP, STACK, EXACT, BLOCKS>, dim3(kSms * BLOCKS), dim3(32 * FewCfg<DP, STACK, BLOCKS>::WARPS), bytes, st, a);
}

// An SM's warps are one block, or several where there are many items: one block's beginnings and ends of items then lie under the others'
// copies.  256 sequences of up to 1000 tokens, 8 heads, 151 us with one block, 98 with three; 64 of up to 16000 254 and 233, in runs
// of a second 283 and 270 (16 rows: 425 and 403 with two).  Fewer items are cut in more parts then.  One block and three at 64, 80, 96,
// 112 and 128 items: of up to 4000 tokens 23.3 24.4, 24.1 24.7, 27.4 26.2, 28.9 28.8, 33.1 30.4 us; of up to 16000 44.6 46.5, 53.1 53.8,
// 60.7 60.2, 70.4 68.8, 74.1 71.6; of up to 300 10.8 12.2, then 15.5 12.2 from 80 items on.  Two blocks for 16 rows lose a little at 96
// (41.5 45.8, 97.7 100.2) and gain from 128 on (51.0 50.5, 121.2 119.2).
constexpr int kManyItems = 96, kMostBlocks = 3;
template <int DP, bool EXACT>
int few(const AttnArgs& a, cudaStream_t st) {
    const bool many = (int64_t)a.seqs * a.heads >= kManyItems;
    if (a.most <= 8) return many ? run_few<DP, true, EXACT, kMostBlocks>(a, st) : run_few<DP, true, EXACT, 1>(a, st);
    return many ? run_few<DP, false, EXACT, 2>(a, st) : run_few<DP, false, EXACT, 1>(a, st);
}
template <int DP>
int few(const AttnArgs& a, cudaStream_t st) {
    return a.dim == DP ? few<DP, true>(a, st) : few<DP, false>(a, st);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
static_assert(kMostBlocks * kSms <= MCU_COUNTERS, "a counter for each block");
constexpr int kFewRows = 16;
int padded(const mcu_attention* a) { return a->cache.head_dim <= 64 ? 64 : 128; }

// The kernels of a call.  Sequences of up to `few` rows of a kv head go to attention_few; the host knows an upper bound of
// new tokens only, so above it the other kernel takes what is longer, and both are launched unless every sequence may have
// the bound (a full rectangle of rows).
struct Forms {
    int few;
    bool tiles;
};
Forms forms_of(const mcu_attention* a) {
    const int64_t group = a->q_heads / a->cache.heads, most = a->max_new * group;
    if (most <= kFewRows) return Forms{most <= 8 ? 8 : kFewRows, false};
    if (a->rows == a->seqs * a->max_new) return Forms{0, true};
    return Forms{group <= 8 ? 8 : group <= kFewRows ? kFewRows : 0, true};
}

// Scratch: the parts of tiles, then those of few rows, then counters for a call that got none.
int64_t few_floats(const mcu_attention* a, const Forms& f) { return f.few ? 2 * kSms * kMostBlocks * part_floats(kFewRows, padded(a)) : 0; }
int64_t tile_floats(const mcu_attention* a, const Forms& f) { return f.tiles ? 2 * kSms * part_floats(kTileRows, padded(a)) : 0; }

}  // namespace

extern "C" size_t mcu_attention_scratch_bytes(const mcu_attention* a) {
    const Forms f = forms_of(a);
    return (size_t)(tile_floats(a, f) + few_floats(a, f) + (f.few ? kMostBlocks * kSms : 0)) * 4;
}

extern "C" int mcu_launch_attention(const mcu_attention* c, void* scratch, uint32_t* joins, int* status, cudaStream_t st, int* launches) {
    const int group = (int)(c->q_heads / c->cache.heads);
    const Forms f = forms_of(c);
    AttnArgs a = {};
    a.out = c->out, a.lse = c->lse, a.q = c->q, a.k = c->cache.k, a.v = c->cache.v, a.ks = c->cache.k_scale, a.vs = c->cache.v_scale;
    a.table = c->table, a.start = c->start, a.length = c->length, a.table_s1 = c->table_s1, a.q_s1 = c->q_s1, a.out_s1 = c->out_s1;
    a.parts = (float*)scratch, a.status = status, a.joins = joins, a.seqs = (int)c->seqs, a.rows = (int)c->rows, a.max_new = (int)c->max_new;
    a.heads = c->cache.heads, a.group = group, a.dim = c->cache.head_dim, a.pages = c->cache.pages;
    while ((1 << a.page_log) < c->cache.page_size) ++a.page_log;
    a.window = c->window >= ((int64_t)1 << 31) - 1 ? 0 : (int)c->window;
    a.longest = (int)(c->table_s1 * c->cache.page_size);
    a.blocks = kSms, a.scale = c->scale, a.stall = test_stall();
    a.q_vec = aligned16(c->q) && !(c->q_s1 & 3), a.out_vec = aligned16(c->out) && !(c->out_s1 & 3);
    const bool wide = a.dim > 64;
    int rc = 0;
    *launches = 0;
    if (f.tiles) {
        a.least = f.few + 1, a.most = 0x7fffffff;
        rc = wide ? run_tiles<128>(a, st) : run_tiles<64>(a, st);
        *launches += 2;
        a.parts += tile_floats(c, f);
    }
    if (!rc && f.few) {
        a.least = 1, a.most = f.few;
        if (!joins) {
            a.joins = (uint32_t*)(a.parts + few_floats(c, f));
            if ((rc = (int)cudaMemsetAsync(a.joins, 0, kMostBlocks * kSms * 4, st))) return rc;
        }
        rc = wide ? few<128>(a, st) : few<64>(a, st);
        *launches += 1;
    }
    return rc;
}
