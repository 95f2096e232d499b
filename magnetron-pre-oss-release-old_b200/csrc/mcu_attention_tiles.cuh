// Attention over the paged e4m3 cache for sequences of many rows (new tokens x query heads of a group).
#ifndef MCU_ATTENTION_TILES_CUH
#define MCU_ATTENTION_TILES_CUH
#include "mcu_attention.cuh"
#include "mcu_tc.cuh"

namespace {

using namespace mcu;

// ------------------------------------------------------------ many rows: chunks and prompts
//
// A block takes tiles of 128 rows of a kv head through their tokens, 128 at a time, on tcgen05.mma kind::f16:
//   S = Qh K^T + Ql K^T,   O = Ph V + Pl V,
// Q and P as two f16 (22 bits), K and V exact in f16.  Both left operands lie in TMEM, where a product's rate does not hang on
// two operands' shared-memory reads: 2 x 128 columns of S, over which P is written in place, 128 of O, 128 of Q.  O starts
// from zero for every 128 tokens and is added in registers in f32 (rounded to nearest), times the step of the row's reference and
// the unit of the tile's value scales: no accumulator is ever rescaled, and the tensor core's truncating sums stay short.
//   warps 0-7    softmax: warp w has the rows 32 (w & 3) .. and half w / 4 of the tokens and of the output's columns
//   warps 8-11   loaders: e4m3 from the pages through registers to f16 tiles (128-byte swizzle), scales, valid tokens
//   warp 12      issues the products: S of tile j + 1 before O of tile j, so that softmax runs under them
//   warp 13      plans: puts the block's items into a ring, so that the others find theirs without global loads
// A tile's logits are read twice, for the rows' maxima and for the probabilities, in loops of 32 columns that are not unrolled:
// the loops of all roles have to fit the SM's instruction cache together (unrolled, with the probabilities formed in one pass
// against a reference that moved when it had to, a third of its requests missed and a tile took three times as long).
constexpr int kTileRows = 128, kTileTokens = 128, kTileThreads = 512;
constexpr int kTileLaunch = 128, kSoftRegs = 168, kLoadRegs = 128, kIssueRegs = 48;
static_assert(2 * kSoftRegs + kLoadRegs + kIssueRegs == 4 * kTileLaunch, "register split must match the launch");
constexpr int kItems = 4;             // items in the planner's ring

// What the roles need of an item, as the planner leaves it; rows = 0: no more.
struct __align__(16) TileItem {
    int rows, n, row0, first_row;        // n: tiles of 128 tokens
    int pos, all_first, all_last, head;  // every row sees the tokens all_first .. all_last
    int low, high, first, seq;           // first: the first token of the first tile
    int whole, begins, last_block, pad;
};
static_assert(sizeof(TileItem) == 64, "four 16-byte pieces");

template <int DP>
struct TileCfg {
    static constexpr int BLOCKS = DP / 64;                   // column blocks of 64 f16
    static constexpr int TILE = BLOCKS * kTileTokens * 128;  // bytes of a K or V tile
    static constexpr int K = 0, V = 2 * TILE;
    static constexpr int SCALES = 4 * TILE;                  // 4 x {keys' scales, values' ratios, valid tokens, unit}
    static constexpr int SLOT = 2 * kTileTokens * 4 + 32;
    static constexpr int MAXIMA = SCALES + 4 * SLOT;         // [2][2][128]
    static constexpr int SUMS = MAXIMA + 2 * 2 * 128 * 4;    // [2][128]
    static constexpr int TOPS = SUMS + 2 * 128 * 4;          // [2][4] of the loaders
    static constexpr int PLACES = TOPS + 32;                 // [8] of the loaders
    static constexpr int ITEMS = PLACES + 64;
    static constexpr int BARS = ITEMS + kItems * 64;
    static constexpr int SMEM = BARS + 256 + 1024;
    static constexpr uint32_t S_COL = 0, O_COL = 256, Q_COL = 384;
    static_assert(Share<kTileRows, DP, kTileThreads>::SMEM <= SCALES, "the search for work takes the tiles' room");
    static_assert(SMEM <= 227 * 1024, "must fit shared memory");
};

__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// The whole warp waits, polled by one lane.  The __syncwarp holds the other lanes back: a shuffle whose result is not
// used does not.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, const Abort& ab, int code) {
    uint32_t ok = 1;
    if ((threadIdx.x & 31) == 0) ok = mbar_wait(bar, parity, ab, code);
    __syncwarp();
    return __shfl_sync(0xffffffffu, ok, 0) != 0;
}
__device__ __forceinline__ void bar_named(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
// A barrier that also says whether any of its threads came with true.
__device__ __forceinline__ bool bar_any(int id, int threads, bool mine) {
    uint32_t any;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %3, 0;\n\t"
        "barrier.cta.red.or.pred q, %1, %2, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(any)
        : "r"(id), "r"(threads), "r"((uint32_t)mine)
        : "memory");
    return any != 0;
}

// D (+)= A B with A (f16) in TMEM; one thread.
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc));
}
// D f32, A and B f16; B with the inner index (0) or the columns (1) along its rows.
__device__ __forceinline__ uint32_t idesc_f16(int n, int b_turned) {
    return (1u << 4) | ((uint32_t)b_turned << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTileRows >> 4) << 24);
}
// A tile of rows of 128 bytes, 128-byte swizzle, 8 rows 1024 bytes; `lead`: bytes between blocks of 64 columns of a turned operand.
__device__ __forceinline__ uint64_t tile_desc(uint32_t saddr, uint32_t lead) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)((lead >> 4) & 0x3FFFu) << 16 | (uint64_t)(1024u >> 4) << 32 | (uint64_t)1 << 46 |
           (uint64_t)2 << 61;
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(v[0]),
        "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]),
        "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st_done() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void sts128(uint32_t a, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// Pairs of f32 in one instruction, each rounded as alone.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ uint64_t pair_of(uint32_t a, uint32_t b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// As split2, for a pair.
__device__ __forceinline__ void split_pair(uint64_t w, uint32_t& high, uint32_t& low) {
    asm("{\n\t.reg .b16 x, y;\n\t.reg .f32 a, b, u, v;\n\t.reg .b64 h, d;\n\t"
        "mov.b64 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.f32 %0, b, a;\n\t"
        "mov.b32 {x, y}, %0;\n\t"
        "cvt.f32.f16 u, x;\n\t"
        "cvt.f32.f16 v, y;\n\t"
        "sub.f32 u, a, u;\n\t"
        "sub.f32 v, b, v;\n\t"
        "cvt.rn.f16x2.f32 %1, v, u;\n\t}"
        : "=&r"(high), "=r"(low)
        : "l"(w));
}

// 32 columns of S to probabilities times their values' ratios, as f16 halves; *sum gains the probabilities.  Tokens that are
// not to be seen have come as -inf.
// CARE: for scales that are no numbers and for logits that are large.  Tokens whose bit in `seen` is not set have no part,
// whatever their scales are, and a logit is rounded before the reference is taken from it, so that the two are equal where they
// should be (unrounded they differ by up to 2^-24 of the logit: of no account while that is small).
template <bool CARE>
__device__ __forceinline__ void tile_chunk(const uint32_t (&v)[32], const ulonglong2* ks, const ulonglong2* vs, float m, uint64_t rf, uint32_t seen,
                                           uint32_t* high, uint32_t* low, uint64_t* sum) {
    const uint64_t top = pair_of(kTop, kTop), minus_m = pair_of(-m, -m);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const ulonglong2 kk = ks[k], vv = vs[k];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int e = 4 * k + 2 * h;
            const uint64_t kp = h ? kk.y : kk.x, vp = h ? vv.y : vv.x;
            float x, y;
            uint64_t t;
            if (CARE) {  // (one by one: packed, the compiler joins the two roundings)
                unpair(kp, x, y);
                t = pair_of(__fadd_rn(__fmul_rn(__uint_as_float(v[e]), x), -m), __fadd_rn(__fmul_rn(__uint_as_float(v[e + 1]), y), -m));
            } else {
                t = fma2(pair_of(v[e], v[e + 1]), kp, minus_m);
            }
            unpair(fma2(t, rf, top), x, y);
            x = exp2_f(x), y = exp2_f(y);
            if (CARE) x = seen >> e & 1 ? x : 0.0f, y = seen >> (e + 1) & 1 ? y : 0.0f;
            const uint64_t p = pair_of(x, y);
            *sum = add2(*sum, p);
            uint64_t w = mul2(p, vp);
            if (CARE) {
                unpair(w, x, y);
                w = pair_of(seen >> e & 1 ? x : 0.0f, seen >> (e + 1) & 1 ? y : 0.0f);
            }
            split_pair(w, high[2 * k + h], low[2 * k + h]);
        }
    }
}

template <int DP>
__global__ void __maxnreg__(kTileLaunch) attention_tiles(AttnArgs a) {
    using C = TileCfg<DP>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 1023u);
    uint64_t* k_full = (uint64_t*)(smem + C::BARS);
    uint64_t* k_empty = k_full + 2;
    uint64_t* v_full = k_empty + 2;
    uint64_t* v_empty = v_full + 2;
    uint64_t* s_full = v_empty + 2;
    uint64_t* p_full = s_full + 2;
    uint64_t* sc_full = p_full + 2;  // four
    uint64_t* o_full = sc_full + 4;
    uint64_t* o_free = o_full + 1;
    uint64_t* q_full = o_free + 1;
    uint64_t* drain = q_full + 1;
    uint64_t* i_full = drain + 1;  // kItems each
    uint64_t* i_free = i_full + kItems;
    uint32_t* tmem_slot = (uint32_t*)(i_free + kItems);
    volatile int* gave_up = (volatile int*)(tmem_slot + 1);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const Abort ab{gave_up, a.status};
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], 128);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_full[i], 128);
            mbar_init(&v_empty[i], 1);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 256);
        }
        for (int i = 0; i < 4; ++i) mbar_init(&sc_full[i], 128);
        for (int i = 0; i < kItems; ++i) {
            mbar_init(&i_full[i], 1);
            mbar_init(&i_free[i], 13);  // a lane of each softmax and loader warp and of the issuer
        }
        mbar_init(o_full, 1);
        mbar_init(o_free, 256);
        mbar_init(q_full, 256);
        mbar_init(drain, 1);
        *gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_begin();
    const uint32_t tmem = *tmem_slot;

    Share<kTileRows, DP, kTileThreads> sh;
    const bool work = sh.find(a, (int64_t*)smem);
    __syncthreads();

    // Item i of the block's, once the planner has it there.  The warps that meet at named barriers (id, threads; 0: none) end
    // together: a barrier tells whether any of them saw that a wait was given up.
    const uint32_t ring = smem_u32(smem + C::ITEMS);
    auto item = [&](uint32_t i, int id, int threads) {
        warp_wait(&i_full[i & (kItems - 1)], i / kItems & 1, ab, 41);
        TileItem it;
        int* w = (int*)&it;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint4 v = ((const uint4*)(smem + C::ITEMS))[4 * (i & (kItems - 1)) + k];
            w[4 * k] = (int)v.x, w[4 * k + 1] = (int)v.y, w[4 * k + 2] = (int)v.z, w[4 * k + 3] = (int)v.w;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&i_free[i & (kItems - 1)]);
        const bool over = *gave_up != 0;
        if (threads ? bar_any(id, threads, over) : __any_sync(0xffffffffu, over)) it.rows = 0;
        return it;
    };

    if (!work) {
        // nothing to do but to free TMEM
    } else if (warp < 8) {  // ---- softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
        constexpr int HD = DP / 2;  // this thread's columns of the output and values of a query
        const int half = warp >> 2, row = 32 * (warp & 3) + lane, pair = 1 + (warp & 3);
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        float* maxima = (float*)(smem + C::MAXIMA);
        float* sums = (float*)(smem + C::SUMS);
        uint32_t t = 0;  // tiles done
        // The item at hand: its rows' reference and sum, output, the factor that takes S to log2 units.
        TileItem it = {};
        uint64_t o[HD / 2];
        float m = -INFINITY, l = 0.0f, rf = 0.0f, fade = 1.0f, unit = 0.0f;
        // O of the last tile joins the sums: waits for it, and hands the columns back
        auto add_tile = [&](uint32_t x) {
            if (__any_sync(0xffffffffu, fade != 1.0f)) {
                const uint64_t f = pair_of(fade, fade);
#pragma unroll
                for (int k = 0; k < HD / 2; ++k) o[k] = mul2(o[k], f);
            }
            const uint64_t u = pair_of(unit, unit);
            warp_wait(o_full, x & 1, ab, 31);
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < HD / 32; ++c) {
                uint32_t v[32];
                tmem_ld32(tmem + lanes + C::O_COL + HD * half + 32 * c, v);
                if (c == HD / 32 - 1) {
                    tc_fence_before();
                    mbar_arrive(o_free);
                }
#pragma unroll
                for (int k = 0; k < 16; ++k) o[16 * c + k] = fma2(pair_of(v[2 * k], v[2 * k + 1]), u, o[16 * c + k]);
            }
        };
#pragma unroll 1
        for (uint32_t i = 0;; ++i) {
            const TileItem next = item(i, pair, 64);
            float next_rf = 0.0f;
            if (next.rows && next.n) {
                // the next item's queries, as two f16 in TMEM (the products that read the last item's are done: their S was
                // waited for), before the last product of the item at hand is waited for
                const int r = next.first_row + row;
                const bool live = row < next.rows;
                const float* p = a.q + (int64_t)(next.row0 + (live ? r / a.group : 0)) * a.q_s1 +
                                 (int64_t)(next.head * a.group + (live ? r % a.group : 0)) * a.dim + HD * half;
                float x[HD];
                uint32_t top = 0;
                if (a.q_vec) {
#pragma unroll
                    for (int k = 0; k < HD / 4; ++k) {
                        const float4 v = live && HD * half + 4 * k < a.dim ? *(const float4*)(p + 4 * k) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        x[4 * k] = v.x, x[4 * k + 1] = v.y, x[4 * k + 2] = v.z, x[4 * k + 3] = v.w;
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < HD; ++k) x[k] = live && HD * half + k < a.dim ? p[k] : 0.0f;
                }
#pragma unroll
                for (int k = 0; k < HD; ++k) top = max(top, abs_bits(x[k]));
                sums[half * 128 + row] = __uint_as_float(top);
                bar_named(pair, 64);
                top = max(top, __float_as_uint(sums[(half ^ 1) * 128 + row]));
                bar_named(pair, 64);
                const float up = query_unit(top);
#pragma unroll
                for (int c = 0; c < HD / 32; ++c) {
                    uint32_t h[16], lo[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) split2(x[32 * c + 2 * k] * up, x[32 * c + 2 * k + 1] * up, h[k], lo[k]);
                    tmem_st16(tmem + lanes + C::Q_COL + HD / 2 * half + 16 * c, h);
                    tmem_st16(tmem + lanes + C::Q_COL + DP / 2 + HD / 2 * half + 16 * c, lo);
                }
                tmem_st_done();
                tc_fence_before();
                mbar_arrive(q_full);
                next_rf = a.scale * kLog2e / up;
            }
            if (it.rows) {  // the item at hand is complete but for its last tile's output
                if (it.n) add_tile(t - 1);
                sums[half * 128 + row] = l;
                bar_named(pair, 64);
                l += sums[(half ^ 1) * 128 + row];
                bar_named(pair, 64);
                if (row < it.rows) {
                    const int r = it.first_row + row;
                    const float k = l == 0.0f ? 0.0f : 0x1p16f / l;  // (units are kept 2^-16 of theirs: no sum of theirs overflows)
                    const float top = m == -INFINITY ? kNone : fmaf(m, rf, -kTop);
                    float* dst;
                    bool vec = true;
                    if (it.whole) {
                        const int head = it.head * a.group + r % a.group;
                        const int64_t token = it.row0 + r / a.group;
                        dst = a.out + token * a.out_s1 + (int64_t)head * a.dim, vec = a.out_vec;
                        if (a.lse && half == 0) a.lse[token * a.heads * a.group + head] = l == 0.0f ? -INFINITY : (top + log2f(l)) * kLn2;
                    } else {
                        float* p = part_slot(a, kTileRows, DP, blockIdx.x, it.begins);
                        dst = p + 8 + 2 * kTileRows + row * DP;
                        if (half == 0) {
                            p[8 + 2 * row] = top, p[9 + 2 * row] = l;
                            if (row == 0 && it.begins) {
                                int* w = (int*)p;
                                w[1] = it.head, w[2] = it.rows, w[3] = it.first_row, w[4] = it.row0, w[5] = it.last_block, w[0] = 1;
                            }
                        }
                    }
                    dst += HD * half;
                    const uint64_t kk = pair_of(k, k);
#pragma unroll
                    for (int c = 0; c < HD / 4; ++c) {
                        float4 v;
                        unpair(mul2(o[2 * c], kk), v.x, v.y);
                        unpair(mul2(o[2 * c + 1], kk), v.z, v.w);
                        if (HD * half + 4 * c >= a.dim) continue;
                        if (vec) {
                            *(float4*)(dst + 4 * c) = v;
                        } else {
                            dst[4 * c] = v.x, dst[4 * c + 1] = v.y, dst[4 * c + 2] = v.z, dst[4 * c + 3] = v.w;
                        }
                    }
                }
            }
            if (!next.rows) break;
            it = next, rf = next_rf;
            const int last = row < it.rows ? it.pos + (it.first_row + row) / a.group : -1;
            const int first = a.window && last >= a.window ? last - a.window + 1 : 0;
            const uint64_t rf2 = pair_of(rf, rf);
#pragma unroll
            for (int k = 0; k < HD / 2; ++k) o[k] = 0;
            m = -INFINITY, l = 0.0f, fade = 1.0f, unit = 0.0f;
            const bool wild = !(rf >= 0x1p-126f);  // a row's logits want the careful form
#pragma unroll 1
            for (int j = 0; j < it.n; ++j, ++t) {
                const uint8_t* slot = smem + C::SCALES + (t & 3) * C::SLOT;
                const ulonglong2* ks = (const ulonglong2*)(slot + 64 * half * 4);
                const ulonglong2* vs = (const ulonglong2*)(slot + (kTileTokens + 64 * half) * 4);
                warp_wait(&sc_full[t & 3], t >> 2 & 1, ab, 32);
                const int j0 = it.first + kTileTokens * j;
                const uint4 ok = *(const uint4*)(slot + 2 * kTileTokens * 4);
                const float2 more = *(const float2*)(slot + 2 * kTileTokens * 4 + 16);  // unit, and 0 where a scale is no number
                // not all tokens seen by all rows
                const bool edge = j0 < it.all_first || j0 + kTileTokens - 1 > it.all_last || (ok.x & ok.y & ok.z & ok.w) != 0xffffffffu;
                uint32_t seen0 = half ? ok.z : ok.x, seen1 = half ? ok.w : ok.y;
                if (edge) {
                    const int lo = first - j0 - 64 * half, hi = last - j0 - 64 * half;  // tokens lo .. hi of this half's
                    const int a0 = max(lo, 0), b0 = min(hi, 31), a1 = max(lo - 32, 0), b1 = min(hi - 32, 31);
                    seen0 &= a0 > b0 ? 0u : (0xffffffffu << a0) & (0xffffffffu >> (31 - b0));
                    seen1 &= a1 > b1 ? 0u : (0xffffffffu << a1) & (0xffffffffu >> (31 - b1));
                }
                warp_wait(&s_full[t & 1], t >> 1 & 1, ab, 33);
                tc_fence_after();
                const uint32_t sc = tmem + lanes + C::S_COL + 128 * (t & 1) + 64 * half;
                // the rows' maxima, of both halves
                float x = -INFINITY;
#pragma unroll 1
                for (int c = 0; c < 2; ++c) {
                    uint32_t v[32];
                    tmem_ld32(sc + 32 * c, v);
                    float y = -INFINITY, z = -INFINITY;
                    const uint32_t seen = c ? seen1 : seen0;
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const ulonglong2 kk = ks[8 * c + k];
                        float p[4];
                        unpair(mul2(pair_of(v[4 * k], v[4 * k + 1]), kk.x), p[0], p[1]);
                        unpair(mul2(pair_of(v[4 * k + 2], v[4 * k + 3]), kk.y), p[2], p[3]);
                        if (edge) {
#pragma unroll
                            for (int q = 0; q < 4; ++q) p[q] = seen >> (4 * k + q) & 1 ? p[q] : -INFINITY;
                        }
                        y = max3(y, p[0], p[1]), z = max3(z, p[2], p[3]);
                    }
                    x = max3(x, y, z);
                }
                maxima[((t & 1) * 2 + half) * 128 + row] = x;
                bar_named(pair, 64);
                x = fmaxf(x, maxima[((t & 1) * 2 + (half ^ 1)) * 128 + row]);
                float step = 1.0f;
                if (x > m) {
                    step = m == -INFINITY ? 0.0f : exp2_f((m - x) * rf);
                    m = x;
                    l *= step;
                }
                const float ref = m == -INFINITY ? 0.0f : m;
                const bool care = __any_sync(0xffffffffu, wild || more.y == 0.0f || !(fabsf(ref * rf) <= 0x1p14f));
                uint64_t sum = 0;
#pragma unroll 1
                for (int c = 0; c < 2; ++c) {
                    uint32_t v[32], h[16], lo[16];
                    tmem_ld32(sc + 32 * c, v);
                    const uint32_t seen = c ? seen1 : seen0;
                    if (care) {
                        tile_chunk<true>(v, ks + 8 * c, vs + 8 * c, ref, rf2, seen, h, lo, &sum);
                    } else {
                        if (edge) {
#pragma unroll
                            for (int k = 0; k < 32; ++k) v[k] = seen >> k & 1 ? v[k] : 0xff800000u;
                        }
                        tile_chunk<false>(v, ks + 8 * c, vs + 8 * c, ref, rf2, 0u, h, lo, &sum);
                    }
                    tmem_st16(sc + 32 * c, h);
                    tmem_st16(sc + 32 * c + 16, lo);
                }
                float y;
                unpair(sum, x, y);
                l += x + y;
                tmem_st_done();
                tc_fence_before();
                mbar_arrive(&p_full[t & 1]);
                if (j) add_tile(t - 1);
                fade = step, unit = more.x;
            }
        }
    } else if (warp < 12) {  // ---- loaders
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLoadRegs));
        constexpr int CH = DP / 16, PER = kTileTokens * CH / 128;  // pieces of 16 bytes of a row, and of a thread
        constexpr int STEP = 128 / CH;                             // rows between a thread's pieces
        // Eight lanes that store 16 bytes each have four pieces of two neighbouring rows, whose places in the swizzle differ by one:
        // no two have the same banks.
        const int tid = threadIdx.x - 256, lw = warp - 8;
        const int ch = CH == 8 ? (lane & 3) | (lane >> 1 & 4) : lane & 3;
        const int r0 = CH == 8 ? 4 * lw + (lane >> 2 & 1) + (lane >> 3 & 2) : 8 * lw + (lane >> 2);
        uint32_t* tops = (uint32_t*)(smem + C::TOPS);
        int64_t* places = (int64_t*)(smem + C::PLACES);
        const uint32_t piece = (uint32_t)(ch >> 2) * (kTileTokens * 128) + r0 * 128;
        uint8_t* at0 = smem + piece + ((2 * (ch & 3)) ^ (r0 & 7)) * 16;
        uint8_t* at1 = smem + piece + ((2 * (ch & 3) + 1) ^ (r0 & 7)) * 16;
        static_assert(STEP % 8 == 0, "a thread's rows have one place in the swizzle");
        if (a.stall) warp_wait(&k_empty[0], 0, ab, 34);  // a test of the bounded waits: nothing completes this phase
        auto put = [&](uint32_t tile, const uint4 (&x)[PER]) {
#pragma unroll
            for (int k = 0; k < PER; ++k) {
                const uint4 v = x[k];
                const uint4 lo = make_uint4(f16_of_e4m3(v.x), f16_of_e4m3(v.x >> 16), f16_of_e4m3(v.y), f16_of_e4m3(v.y >> 16));
                const uint4 hi = make_uint4(f16_of_e4m3(v.z), f16_of_e4m3(v.z >> 16), f16_of_e4m3(v.w), f16_of_e4m3(v.w >> 16));
                *(uint4*)(at0 + tile + k * (STEP * 128)) = lo;
                *(uint4*)(at1 + tile + k * (STEP * 128)) = hi;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        };
        uint4 kv[PER], vv[PER];
        float ks = 0.0f, vs = 0.0f;
        bool in = false;
        TileItem it = {};
        int j = -1;          // the tile of the item that the registers are filled for
        int page = -1;       // lane g & 7: the page of group g (16 tokens) of the tile after
        uint32_t rows = 0;   // of the thread's pieces, those that exist
        bool some = false;   // not all of the warp's do
        auto look = [&](int x) {
            const int at = it.first + kTileTokens * x + 16 * (lane & 7);
            page = x < it.n && at < it.high ? a.table[(int64_t)it.seq * a.table_s1 + (at >> a.page_log)] : -1;
        };
        // (a piece that does not exist is read from the cache's first slot and cleared)
        const int64_t own = (int64_t)(r0 & 15) * a.dim + (16 * ch < a.dim ? 16 * ch : 0);
        auto fetch = [&](const uint8_t* from, uint4 (&to)[PER]) {
            from += own;
#pragma unroll
            for (int k = 0; k < PER; ++k) to[k] = __ldg((const uint4*)(from + places[(STEP * k + r0) >> 4]));
            if (some) {
#pragma unroll
                for (int k = 0; k < PER; ++k)
                    if (!(rows >> k & 1)) to[k] = make_uint4(0, 0, 0, 0);
            }
        };
        // Tile t goes from registers to shared memory, each half followed by the loads of the next tile's, which may be another
        // item's.
        bool have = false, more = true;
        uint32_t items = 0;
#pragma unroll 1
        for (uint32_t t = 0; more || have;) {
            if (have) {
                // scales: the unit is the least power of two above the tile's largest
                const bool number = vs < kLargestScale;
                float top = number ? vs : 0.0f;
#pragma unroll
                for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                const uint32_t bits = __ballot_sync(0xffffffffu, in);
                const bool bad = __any_sync(0xffffffffu, !number || !(fabsf(ks) < INFINITY));
                if (lane == 0) tops[(t & 1) * 4 + lw] = abs_bits(top) | (bad ? 0x80000000u : 0u);
                warp_wait(&k_empty[t & 1], (t >> 1 & 1) ^ 1, ab, 34);
                bar_named(5, 128);
                const uint4 all = *(const uint4*)(tops + (t & 1) * 4);
                const uint32_t largest = max(max(all.x & 0x7FFFFFFFu, all.y & 0x7FFFFFFFu), max(all.z & 0x7FFFFFFFu, all.w & 0x7FFFFFFFu));
                const float unit = unit_above(fmaxf(__uint_as_float(largest), kLeastUnit));
                float* slot = (float*)(smem + C::SCALES + (t & 3) * C::SLOT);
                slot[tid] = ks == 0.0f ? 0x1p-126f : ks;  // (so that -inf times it is -inf)
                slot[kTileTokens + tid] = vs * (1.0f / unit);
                if (lane == 0) slot[2 * kTileTokens + lw] = __uint_as_float(bits);
                if (tid == 0) slot[2 * kTileTokens + 4] = unit * 0x1p-16f, slot[2 * kTileTokens + 5] = (all.x | all.y | all.z | all.w) >> 31 ? 0.0f : 1.0f;
                mbar_arrive(&sc_full[t & 3]);
                put(C::K + (t & 1) * C::TILE, kv);
                mbar_arrive(&k_full[t & 1]);
            }
            // the next tile
            ++j;
            if (j >= it.n) {
                do {
                    it = item(items++, 5, 128);
                } while (it.rows && !it.n);
                more = it.rows != 0;
                j = 0;
                look(0);
            }
            if (more) {
                const int tok = it.first + kTileTokens * j;
                const bool exists = (uint32_t)page < (uint32_t)a.pages;
                const int at = tok + 16 * (lane & 7);
                const int64_t slot0 = exists ? ((((int64_t)page * a.heads) + it.head) << a.page_log) + (at & ((1 << a.page_log) - 1)) : (int64_t)0;
                bar_named(5, 128);  // (the last tile's places have been read)
                if (lw == 0 && lane < 8) places[lane] = slot0 * a.dim;
                const uint32_t groups = __ballot_sync(0xffffffffu, exists) & 0xffu;
                const int64_t s = __shfl_sync(0xffffffffu, slot0, tid >> 4) + (tid & 15);
                in = (groups >> (tid >> 4) & 1) && tok + tid >= it.low && tok + tid < it.high;
                ks = __ldg(a.ks + s), vs = __ldg(a.vs + s);
                if (!in) ks = vs = 0.0f;
                some = groups != 0xffu || tok < it.low || tok + kTileTokens > it.high || a.dim != DP;
                if (some) {
                    rows = 0;
#pragma unroll
                    for (int k = 0; k < PER; ++k) {
                        const int r = STEP * k + r0;
                        rows |= (uint32_t)((groups >> (r >> 4) & 1) && tok + r >= it.low && tok + r < it.high && 16 * ch < a.dim) << k;
                    }
                }
                look(j + 1);
                bar_named(5, 128);
                fetch(a.k, kv);
            }
            if (have) {
                warp_wait(&v_empty[t & 1], (t >> 1 & 1) ^ 1, ab, 35);
                put(C::V + (t & 1) * C::TILE, vv);
                mbar_arrive(&v_full[t & 1]);
                ++t;
            }
            if (more) fetch(a.v, vv);
            have = more;
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
        if (warp == 12) {  // ---- issuer
            const int steps = a.dim / 16;
            const uint32_t is = idesc_f16(kTileTokens, 0), io = idesc_f16(a.dim, 1);
            const uint64_t k0 = tile_desc(smem_u32(smem + C::K), 16), v0 = tile_desc(smem_u32(smem + C::V), kTileTokens * 128);
            uint32_t t = 0, queries = 0;
            bool ok = true;
            auto logits = [&](uint32_t x) {
                ok = ok && warp_wait(&k_full[x & 1], x >> 1 & 1, ab, 36);
                tc_fence_after();
                if (ok && elect_one()) {
                    const uint32_t d = tmem + C::S_COL + 128 * (x & 1);
                    const uint64_t b = k0 + (uint64_t)((x & 1) * (C::TILE >> 4));
                    for (int h = 0; h < 2; ++h)
                        for (int s = 0; s < steps; ++s)
                            umma_ts(d, tmem + C::Q_COL + h * (DP / 2) + 8 * s, b + (s >> 2) * ((kTileTokens * 128) >> 4) + (s & 3) * 2, is, h + s);
                    umma_commit(&s_full[x & 1]);
                    umma_commit(&k_empty[x & 1]);
                }
                __syncwarp();
            };
            for (uint32_t i = 0; ok; ++i) {
                const TileItem it = item(i, 0, 0);
                if (!it.rows) break;
                if (!it.n) continue;
                ok = warp_wait(q_full, queries++ & 1, ab, 37);
                tc_fence_after();
                logits(t);
                for (int j = 0; ok && j < it.n; ++j, ++t) {
                    if (j + 1 < it.n) logits(t + 1);
                    ok = ok && warp_wait(&v_full[t & 1], t >> 1 & 1, ab, 38);
                    ok = ok && warp_wait(&p_full[t & 1], t >> 1 & 1, ab, 39);
                    ok = ok && (t == 0 || warp_wait(o_free, (t - 1) & 1, ab, 40));
                    tc_fence_after();
                    if (ok && elect_one()) {
                        const uint32_t p = tmem + C::S_COL + 128 * (t & 1);
                        const uint64_t b = v0 + (uint64_t)((t & 1) * (C::TILE >> 4));
                        for (int h = 0; h < 2; ++h)
                            for (int s = 0; s < 8; ++s)
                                umma_ts(tmem + C::O_COL, p + 32 * (s >> 1) + 8 * (s & 1) + 16 * h, b + s * (2048 >> 4), io, h + s);
                        umma_commit(&v_empty[t & 1]);
                        umma_commit(o_full);
                    }
                    __syncwarp();
                }
            }
            // products in flight end before TMEM is freed
            if (elect_one()) umma_commit(drain);
            __syncwarp();
            if (lane == 0)
                for (uint32_t i = 0; i < kWaitLimit && !mbar_test(drain, 0); ++i) __nanosleep(64);
            __syncwarp();
        } else if (warp == 13) {  // ---- planner
            for (uint32_t i = 0;; ++i) {
                TileItem p = {};
                const bool more = sh.more();
                if (more) {
                    const Item it = sh.item(a);
                    p.rows = it.rows, p.row0 = it.row0, p.first_row = it.first_row;
                    p.n = max(0, min(it.to, (it.high - it.base + kTileTokens - 1) / kTileTokens) - it.from);
                    p.pos = it.pos, p.all_first = it.top_first, p.all_last = it.pos + it.first_row / a.group, p.head = it.head;
                    p.low = it.low, p.high = it.high, p.first = it.base + kTileTokens * it.from, p.seq = it.seq;
                    p.whole = it.from == 0 && it.to == it.units, p.begins = it.from == 0, p.last_block = sh.last_block(it);
                    sh.advance(a, it);
                }
                const bool ok = warp_wait(&i_free[i & (kItems - 1)], (i / kItems & 1) ^ 1, ab, 42);
                if (lane == 0) {
                    const int* w = (const int*)&p;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        sts128(ring + (i & (kItems - 1)) * 64 + 16 * k,
                               make_uint4((uint32_t)w[4 * k], (uint32_t)w[4 * k + 1], (uint32_t)w[4 * k + 2], (uint32_t)w[4 * k + 3]));
                    mbar_arrive(&i_full[i & (kItems - 1)]);
                }
                __syncwarp();
                if (!ok || !more) break;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 12) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
    }
}

template <int DP>
int run_tiles(const AttnArgs& a, cudaStream_t st) {
    static bool done[64];
    const cudaError_t e = allow_smem(attention_tiles<DP>, TileCfg<DP>::SMEM, done);
    if (e != cudaSuccess) return (int)e;
    const int rc = (int)launch_dep(attention_tiles<DP>, dim3((unsigned)a.blocks), dim3(kTileThreads), TileCfg<DP>::SMEM, st, a);
    if (rc) return rc;
    return (int)launch_dep(attention_join<kTileRows, DP>, dim3((unsigned)a.blocks, kTileRows / 4), dim3(128), 0, st, a);
}

}  // namespace
#endif
