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
// from zero for every 128 tokens and is added in registers in f32 (rounded to nearest), times the step of the running maximum and
// the unit of the tile's value scales: no accumulator is ever rescaled, and the tensor core's truncating sums stay short.
//   warps 0-7    softmax: warp w has the rows 32 (w & 3) .. and half w / 4 of the tokens and of the output's columns
//   warps 8-11   loaders: e4m3 from the pages through registers to f16 tiles (128-byte swizzle), scales, valid tokens
//   warp 12      issues the products: S of tile j + 1 before O of tile j, so that softmax runs under them
constexpr int kTileRows = 128, kTileTokens = 128, kTileThreads = 512;
constexpr int kTileLaunch = 128, kSoftRegs = 176, kLoadRegs = 112, kIssueRegs = 48;
static_assert(2 * kSoftRegs + kLoadRegs + kIssueRegs == 4 * kTileLaunch, "register split must match the launch");

template <int DP>
struct TileCfg {
    static constexpr int BLOCKS = DP / 64;                  // column blocks of 64 f16
    static constexpr int TILE = BLOCKS * kTileTokens * 128;  // bytes of a K or V tile
    static constexpr int K = 0, V = 2 * TILE;
    static constexpr int SCALES = 4 * TILE;                  // 4 x {keys' scales, values' ratios, valid tokens, unit}
    static constexpr int SLOT = 2 * kTileTokens * 4 + 32;
    static constexpr int MAXIMA = SCALES + 4 * SLOT;         // [2][2][128]
    static constexpr int SUMS = MAXIMA + 2 * 2 * 128 * 4;    // [2][128]
    static constexpr int TOPS = SUMS + 2 * 128 * 4;          // [2][4] of the loaders
    static constexpr int BARS = TOPS + 32;
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

__device__ __forceinline__ void tmem_load32(uint32_t taddr, float (&v)[32]) {
    uint32_t u[32];
    tmem_ld32(taddr, u);
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(u[i]);
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(v[0]),
        "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]),
        "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st_done() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float4 lds128f(uint32_t a) {
    const uint4 v = lds128(a);
    return make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
}
__device__ __forceinline__ void sts128(uint32_t a, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ float lds32(uint32_t a) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void sts32(uint32_t a, float v) { asm volatile("st.shared.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory"); }

// 128 tokens of an item: how many of its units hold any.
__device__ __forceinline__ int item_tiles(const Item& it) {
    return max(0, min(it.to, (it.high - it.base + kTileTokens - 1) / kTileTokens) - it.from);
}

template <int DP>
__global__ void __maxnreg__(kTileLaunch) attention_tiles(AttnArgs a) {
    using C = TileCfg<DP>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
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
    uint32_t* tmem_slot = (uint32_t*)(drain + 1);
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

    if (!work) {
        // nothing to do but to free TMEM
    } else if (warp < 8) {  // ---- softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
        constexpr int HD = DP / 2;  // this thread's columns of the output and values of a query
        const int half = warp >> 2, row = 32 * (warp & 3) + lane, pair = 1 + (warp & 3);
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t scales = smem_u32(smem + C::SCALES), maxima = smem_u32(smem + C::MAXIMA), sums = smem_u32(smem + C::SUMS);
        uint32_t t = 0;  // tiles done
        while (sh.more()) {
            const Item it = sh.item(a);
            const int n = item_tiles(it), r = it.first_row + row;
            const bool live = row < it.rows;
            float rf = 0.0f;
            if (n) {  // the query's half row, in TMEM as two f16 (products that read the last item's are done: their S was waited for)
                const float* p = a.q + (int64_t)(it.row0 + (live ? r / a.group : 0)) * a.q_s1 +
                                 (int64_t)(it.head * a.group + (live ? r % a.group : 0)) * a.dim + HD * half;
                float x[HD];
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < HD / 4; ++i) {
                    const float4 v = live && HD * half + 4 * i < a.dim ? load4(p + 4 * i, a.q_vec) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    x[4 * i] = v.x, x[4 * i + 1] = v.y, x[4 * i + 2] = v.z, x[4 * i + 3] = v.w;
                }
#pragma unroll
                for (int i = 0; i < HD; ++i) top = max(top, abs_bits(x[i]));
                sts32(sums + (half * 128 + row) * 4, __uint_as_float(top));
                bar_named(pair, 64);
                top = max(top, __float_as_uint(lds32(sums + ((half ^ 1) * 128 + row) * 4)));
                const float up = query_unit(top);
                rf = a.scale * kLog2e / up;
#pragma unroll
                for (int i = 0; i < HD / 32; ++i) {
                    uint32_t h[16], l[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) split2(x[32 * i + 2 * k] * up, x[32 * i + 2 * k + 1] * up, h[k], l[k]);
                    tmem_st16(tmem + lanes + C::Q_COL + HD / 2 * half + 16 * i, h);
                    tmem_st16(tmem + lanes + C::Q_COL + DP / 2 + HD / 2 * half + 16 * i, l);
                }
                tmem_st_done();
                tc_fence_before();
                mbar_arrive(q_full);
            }
            const int last = live ? it.pos + r / a.group : -1, first = a.window && last >= a.window ? last - a.window + 1 : 0;
            const int all_last = it.pos + it.first_row / a.group, all_first = it.top_first;
            float o[HD];
#pragma unroll
            for (int i = 0; i < HD; ++i) o[i] = 0.0f;
            float m = -INFINITY, l = 0.0f, fade = 1.0f, unit = 0.0f;
            // O of tile x joins the sums: waits for it, and hands the columns back
            auto add = [&](uint32_t x) {
                warp_wait(o_full, x & 1, ab, 31);
                tc_fence_after();
                float v[32];
#pragma unroll
                for (int i = 0; i < HD / 32; ++i) {
                    tmem_load32(tmem + lanes + C::O_COL + HD * half + 32 * i, v);
                    if (i == HD / 32 - 1) {
                        tc_fence_before();
                        mbar_arrive(o_free);
                    }
#pragma unroll
                    for (int k = 0; k < 32; ++k) o[32 * i + k] = fmaf(v[k], unit, o[32 * i + k] * fade);
                }
            };
            for (int j = 0; j < n; ++j, ++t) {
                const uint32_t slot = scales + (t & 3) * C::SLOT;
                const int j0 = it.base + kTileTokens * (it.from + j) + 64 * half;
                warp_wait(&sc_full[t & 3], t >> 2 & 1, ab, 32);
                warp_wait(&s_full[t & 1], t >> 1 & 1, ab, 33);
                tc_fence_after();
                const uint32_t sc = tmem + lanes + C::S_COL + 128 * (t & 1) + 64 * half;
                float s[64];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float v[32];
                    tmem_load32(sc + 32 * i, v);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const float4 ks = lds128f(slot + (64 * half + 32 * i + 4 * k) * 4);
                        s[32 * i + 4 * k] = v[4 * k] * ks.x, s[32 * i + 4 * k + 1] = v[4 * k + 1] * ks.y;
                        s[32 * i + 4 * k + 2] = v[4 * k + 2] * ks.z, s[32 * i + 4 * k + 3] = v[4 * k + 3] * ks.w;
                    }
                }
                // valid tokens of the tile, and whether every row sees them all
                const uint4 ok = lds128(slot + 2 * kTileTokens * 4);
                const int tile0 = j0 - 64 * half;
                const bool edge = tile0 < all_first || tile0 + kTileTokens - 1 > all_last || (ok.x & ok.y & ok.z & ok.w) != 0xffffffffu;
                uint32_t seen[2] = {0xffffffffu, 0xffffffffu};
                if (edge) {
#pragma unroll
                    for (int w = 0; w < 2; ++w) {  // tokens first .. last of the 32 from j0 + 32 w
                        const int lo = max(first - j0 - 32 * w, 0), hi = min(last - j0 - 32 * w, 31);
                        const uint32_t range = lo > hi ? 0u : (0xffffffffu << lo) & (0xffffffffu >> (31 - hi));
                        seen[w] = range & (half ? (w ? ok.w : ok.z) : (w ? ok.y : ok.x));
                    }
#pragma unroll
                    for (int k = 0; k < 64; ++k)
                        if (!(seen[k >> 5] >> (k & 31) & 1)) s[k] = -INFINITY;
                }
                float x0 = -INFINITY, x1 = -INFINITY, x2 = -INFINITY, x3 = -INFINITY;
#pragma unroll
                for (int k = 0; k < 64; k += 4) x0 = fmaxf(x0, s[k]), x1 = fmaxf(x1, s[k + 1]), x2 = fmaxf(x2, s[k + 2]), x3 = fmaxf(x3, s[k + 3]);
                float x = fmaxf(fmaxf(x0, x1), fmaxf(x2, x3));
                sts32(maxima + (((t & 1) * 2 + half) * 128 + row) * 4, x);
                bar_named(pair, 64);
                x = fmaxf(x, lds32(maxima + (((t & 1) * 2 + (half ^ 1)) * 128 + row) * 4));
                float step = 1.0f;
                if (x > m) {
                    step = m == -INFINITY ? 0.0f : exp2_f((m - x) * rf);
                    m = x;
                    l *= step;
                }
                const float next_unit = lds32(slot + 2 * kTileTokens * 4 + 16);
                float l0 = 0.0f, l1 = 0.0f;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t h[16], lo[16];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const float4 vs = lds128f(slot + (kTileTokens + 64 * half + 32 * i + 4 * k) * 4);
                        float p[4], w[4];
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            p[q] = exp2_f(fmaf(s[32 * i + 4 * k + q] - m, rf, kTop));
                            if (edge && !(seen[i] >> (4 * k + q) & 1)) p[q] = 0.0f;
                        }
                        l0 += p[0] + p[1], l1 += p[2] + p[3];
                        w[0] = p[0] * vs.x, w[1] = p[1] * vs.y, w[2] = p[2] * vs.z, w[3] = p[3] * vs.w;
                        if (edge) {
#pragma unroll
                            for (int q = 0; q < 4; ++q)
                                if (!(seen[i] >> (4 * k + q) & 1)) w[q] = 0.0f;
                        }
                        split2(w[0], w[1], h[2 * k], lo[2 * k]);
                        split2(w[2], w[3], h[2 * k + 1], lo[2 * k + 1]);
                    }
                    tmem_st16(sc + 32 * i, h);
                    tmem_st16(sc + 32 * i + 16, lo);
                }
                l += l0 + l1;
                tmem_st_done();
                tc_fence_before();
                mbar_arrive(&p_full[t & 1]);
                if (j) add(t - 1);
                fade = step, unit = next_unit;
            }
            if (n) add(t - 1);
            sts32(sums + (half * 128 + row) * 4, l);
            bar_named(pair, 64);
            l += lds32(sums + ((half ^ 1) * 128 + row) * 4);
            bar_named(pair, 64);
            if (live) {
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                const float k = inv * 0x1p15f;
#pragma unroll
                for (int i = 0; i < HD / 4; ++i)
                    if (HD * half + 4 * i < a.dim)
                        put_out(a, sh, it, row, HD * half + 4 * i, make_float4(o[4 * i] * k, o[4 * i + 1] * k, o[4 * i + 2] * k, o[4 * i + 3] * k), top_of(m, rf), l);
            }
            sh.advance(a, it);
        }
    } else if (warp < 12) {  // ---- loaders
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLoadRegs));
        constexpr int CH = DP / 16, PER = kTileTokens * CH / 128;  // pieces of 16 bytes of a row, and of a thread
        constexpr int STEP = 128 / CH;                             // rows between a thread's pieces
        const int tid = threadIdx.x - 256, r0 = tid / CH, ch = tid % CH, lw = warp - 8;
        const uint32_t kt = smem_u32(smem + C::K), vt = smem_u32(smem + C::V), scales = smem_u32(smem + C::SCALES);
        const uint32_t tops = smem_u32(smem + C::TOPS);
        const uint32_t first_at = (uint32_t)(ch >> 2) * (kTileTokens * 128);
        uint32_t t = 0;
        if (a.stall) warp_wait(&k_empty[0], 0, ab, 34);  // a test of the bounded waits: nothing completes this phase
        // 16 bytes of e4m3 to two pieces of f16, that of the other parity first where another lane of the row stores the same banks
        auto put = [&](uint32_t tile, int row, uint4 v) {
            const uint32_t b[4] = {v.x, v.y, v.z, v.w};
            uint32_t f[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) f[2 * i] = f16_of_e4m3(b[i]), f[2 * i + 1] = f16_of_e4m3(b[i] >> 16);
            const uint4 lo = make_uint4(f[0], f[1], f[2], f[3]), hi = make_uint4(f[4], f[5], f[6], f[7]);
            const int odd = ch >> 2 & 1, c0 = 2 * (ch & 3);
            const uint32_t at = tile + first_at + row * 128;
            sts128(at + ((c0 + odd) ^ (row & 7)) * 16, odd ? hi : lo);
            sts128(at + ((c0 + 1 - odd) ^ (row & 7)) * 16, odd ? lo : hi);
        };
        while (sh.more()) {
            const Item it = sh.item(a);
            const int n = item_tiles(it);
            const int32_t* table = a.table + (int64_t)it.seq * a.table_s1;
            uint4 kv[PER], vv[PER];
            float ks = 0.0f, vs = 0.0f;
            bool in = false;
            int pages = -1;  // lane g: the page of group g (16 tokens) of the tile to load
            auto look = [&](int j) {
                const int at = it.base + kTileTokens * (it.from + j) + 16 * (lane & 7);
                pages = j < n && at < it.high ? table[at >> a.page_log] : -1;
            };
            // the slot of row `row` of tile j and whether it has one that any row of the item sees
            auto where = [&](int j, int row, bool& there) {
                const int tok = it.base + kTileTokens * (it.from + j) + row;
                const int pg = __shfl_sync(0xffffffffu, pages, row >> 4);
                there = (uint32_t)pg < (uint32_t)a.pages && tok >= it.low && tok < it.high;
                return there ? (((((int64_t)pg * a.heads) + it.head) << a.page_log) + (tok & ((1 << a.page_log) - 1))) : (int64_t)0;
            };
            auto fetch = [&](int j, const uint8_t* from, uint4 (&to)[PER]) {
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    bool there;
                    const int64_t at = where(j, r0 + STEP * i, there);
                    to[i] = there && 16 * ch < a.dim ? __ldg((const uint4*)(from + at * a.dim + 16 * ch)) : make_uint4(0, 0, 0, 0);
                }
            };
            auto fetch_scales = [&](int j) {
                const int64_t at = where(j, tid, in);
                ks = in ? __ldg(a.ks + at) : 0.0f, vs = in ? __ldg(a.vs + at) : 0.0f;
            };
            if (n) {
                look(0);
                fetch(0, a.k, kv);
                fetch_scales(0);
                fetch(0, a.v, vv);
            }
            for (int j = 0; j < n; ++j, ++t) {
                look(j + 1);
                // scales: the unit is the least power of two above the tile's largest
                const bool number = vs < kLargestScale;
                float top = number ? vs : 0.0f;
#pragma unroll
                for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                const uint32_t bits = __ballot_sync(0xffffffffu, in);
                if (lane == 0) sts32(tops + ((t & 1) * 4 + lw) * 4, top);
                warp_wait(&k_empty[t & 1], (t >> 1 & 1) ^ 1, ab, 34);
                bar_named(5, 128);
                const float4 all = lds128f(tops + (t & 1) * 16);
                const float unit = unit_above(fmaxf(fmaxf(fmaxf(all.x, all.y), fmaxf(all.z, all.w)), kLeastUnit));
                const uint32_t slot = scales + (t & 3) * C::SLOT;
                sts32(slot + tid * 4, ks);
                sts32(slot + (kTileTokens + tid) * 4, vs * (1.0f / unit));
                if (lane == 0) sts32(slot + (2 * kTileTokens + lw) * 4, __uint_as_float(bits));
                if (tid == 0) sts32(slot + (2 * kTileTokens + 4) * 4, unit * 0x1p-15f);
                mbar_arrive(&sc_full[t & 3]);
#pragma unroll
                for (int i = 0; i < PER; ++i) put(kt + (t & 1) * C::TILE, r0 + STEP * i, kv[i]);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(&k_full[t & 1]);
                if (j + 1 < n) {
                    fetch(j + 1, a.k, kv);
                    fetch_scales(j + 1);
                }
                warp_wait(&v_empty[t & 1], (t >> 1 & 1) ^ 1, ab, 35);
#pragma unroll
                for (int i = 0; i < PER; ++i) put(vt + (t & 1) * C::TILE, r0 + STEP * i, vv[i]);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(&v_full[t & 1]);
                if (j + 1 < n) fetch(j + 1, a.v, vv);
            }
            sh.advance(a, it);
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
        if (warp == 12) {  // ---- issuer
            const int steps = (a.dim + 15) / 16;
            const uint32_t is = idesc_f16(kTileTokens, 0), io = idesc_f16(a.dim, 1);
            const uint64_t k0 = tile_desc(smem_u32(smem + C::K), 16), v0 = tile_desc(smem_u32(smem + C::V), kTileTokens * 128);
            uint32_t t = 0, items = 0;
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
            while (ok && sh.more()) {
                const Item it = sh.item(a);
                const int n = item_tiles(it);
                if (n) {
                    ok = warp_wait(q_full, items++ & 1, ab, 37);
                    tc_fence_after();
                    logits(t);
                    for (int j = 0; ok && j < n; ++j, ++t) {
                        if (j + 1 < n) logits(t + 1);
                        ok = ok && warp_wait(&v_full[t & 1], t >> 1 & 1, ab, 38);
                        ok = ok && warp_wait(&p_full[t & 1], t >> 1 & 1, ab, 39);
                        ok = ok && (t == 0 || warp_wait(o_free, (t - 1) & 1, ab, 40));
                        tc_fence_after();
                        if (ok && elect_one()) {
                            const uint32_t p = tmem + C::S_COL + 128 * (t & 1);
                            const uint64_t b = v0 + (uint64_t)((t & 1) * (C::TILE >> 4));
                            for (int h = 0; h < 2; ++h)
#pragma unroll
                                for (int s = 0; s < 8; ++s)
                                    umma_ts(tmem + C::O_COL, p + 32 * (s >> 1) + 8 * (s & 1) + 16 * h, b + s * (2048 >> 4), io, h + s);
                            umma_commit(&v_empty[t & 1]);
                            umma_commit(o_full);
                        }
                        __syncwarp();
                    }
                }
                sh.advance(a, it);
            }
            // products in flight end before TMEM is freed
            if (elect_one()) umma_commit(drain);
            __syncwarp();
            if (lane == 0)
                for (uint32_t i = 0; i < kWaitLimit && !mbar_test(drain, 0); ++i) __nanosleep(64);
            __syncwarp();
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
