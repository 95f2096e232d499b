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
// Q and P (probability times the value's scale) as two f16 (22 bits), K and V exact in f16.  Both left operands lie in TMEM, where a product's rate does not hang on
// two operands' shared-memory reads: 2 x 128 columns of S, over which P is written in place, 128 of O, 128 of Q.  O starts
// from zero for every 128 tokens and is added in registers in f32 (rounded to nearest), times the step from the tile's highest logit
// to the row's and the unit of the tile's value scales: no accumulator is ever rescaled, and the tensor core's truncating sums stay short.
//   warps 0-7    softmax: warp w has the rows 32 (w & 3) .. and half w / 4 of the tokens
//   warps 8-11   sums: O of each tile, in turn, to the rows' f32 sums in registers; the output at the end
//   warps 12-15  loaders: e4m3 from the pages by cp.async, two tiles ahead, then to f16 tiles (128-byte swizzle)
//   warp 16      issues the products: S of tile j + 1 before O of tile j
//   warp 17      plans: puts the block's items into a ring, so that the others find theirs without global loads
//   warp 18      guides: each tile's places in the pages and its scales, up to four tiles ahead; tokens of very different scales of
//                values go into tiles of their own
// What bounds it is the softmax: about 14 instructions for two logits (390 cycles for 32 x 32 of them with four warps a
// scheduler, alone), more than the products' 2 x 1024 cycles a tile.  The loops of all roles have to fit the SM's instruction cache
// together: unrolled for 128 columns they took three times as long.  Eight softmax warps hold half a row's logits each in registers
// (when that was tried, chunks of 300 over 20000 tokens took 214 us; sixteen that read them twice from TMEM 245; two groups of eight in
// turn on tiles of their own more than either).  A unit for each row, found from its weights before they are split, was tried for tiles of
// wide scales: a branch of 220 instructions that no call took made chunks 228 us and prompts 1104, so that such tiles go round instead.  Writing the next item's queries under the last tile's softmax made the loops longer than it hid (prompts
// 1205 us), and fetching them to L2 ahead moved nothing (1059).
// Measured: four prompts of up to 4100 tokens, 32 query heads on 8 of 128: 0.95 ms (0.90 in runs of some milliseconds, before the clock
// falls), 0.37 PFLOP/s (both halves' products 0.75); three chunks of up to 300 over 20000 tokens, 20 heads on 4 of 96: 200 us (196).
constexpr int kTileRows = 128, kTileTokens = 128, kTileThreads = 640;
constexpr int kSoftWarps = 8, kLoadWarp = 12, kIssueWarp = 16, kPlanWarp = 17, kGuideWarp = 18;  // (sums from kSoftWarps on)
constexpr int kTileLaunch = 96, kSoftRegs = 104, kSumRegs = 168, kLoadRegs = 56, kIssueRegs = 48;
static_assert(kSoftRegs >= kTileLaunch && kSumRegs >= kTileLaunch && kLoadRegs <= kTileLaunch && kIssueRegs <= kTileLaunch, "inc or dec as the code has it");
static_assert(2 * kSoftRegs + kSumRegs + kLoadRegs + kIssueRegs == 5 * kTileLaunch, "register split must match the launch");
constexpr int kSoftThreads = 32 * kSoftWarps;
constexpr float kLeastBase = 0x1p-78f;  // unit of a row's sums
// Scales that may share a unit.  A row's largest weight of a tile is at least 2^15 kNear then, and each weight is off by 2^-25 at most (half
// of f16's least step): 128 of them by 2^-33 / kNear of the largest, half an f32 step of it.
constexpr float kNear = 0x1p-8f;
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
    static constexpr int RAW = 4 * TILE;                     // [2] of keys, then values, as loaded: each thread's own pieces
    static constexpr int RAW_TILE = TILE / 2;
    static constexpr int SCALES = RAW + 4 * RAW_TILE;        // 4 x {keys' scales, values' ratios, valid tokens, {unit, item's last, first token}}
    static constexpr int SLOT = 2 * kTileTokens * 4 + 32;
    static constexpr int MAXIMA = SCALES + 4 * SLOT;         // [2][2][128]: of a tile's logits, by half
    static constexpr int SUMS = MAXIMA + 2 * 2 * 128 * 4;    // [2][128]: queries' maxima, by half
    static constexpr int REFS = SUMS + 2 * 128 * 4;          // [4][128] of (the row's maximum, unit): what a tile's O is relative to; the unit below zero: the item's last
    static constexpr int FACTORS = REFS + 4 * 128 * 8;       // [4][128]: rf of an item's rows
    static constexpr int STATS = FACTORS + 4 * 128 * 4;      // [2][128]: an item's sums, by half
    static constexpr int PLACES = STATS + 2 * 128 * 4;   // 4 x {8 groups' offsets in the pages, valid tokens}
    static constexpr int PLACE = 8 * 8 + 16;
    static constexpr int ITEMS = PLACES + 4 * PLACE;
    static constexpr int BARS = ITEMS + kItems * 64;
    static constexpr int SMEM = BARS + 512 + 1024;
    static constexpr uint32_t S_COL = 0, O_COL = 256, Q_COL = 384;
    static_assert(Share<kTileRows, DP, kTileThreads>::SMEM <= RAW, "the search for work takes the tiles' room");
    static_assert(SMEM <= 227 * 1024, "must fit shared memory");
};

__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// The whole warp waits, for about half a second or until a wait was given up elsewhere; the flag then holds the code of a wait that
// was, which goes to the status word when the block ends.  A loop of few instructions: it stands at some twenty places, whose size
// shows in instruction fetches (with the status word written here prompts took 1015 us, 936 so).  A look that finds nothing holds the warp for some 4 us (measured; it ends as soon as there is something), so
// the limit is 2^17 looks; were they to return at once it would be 3 ms, still a hundred times what a tile takes.  The planner, which
// waits for whole items and whose wait is never the first to be given up, has more.  NAP: how many ns to sleep between two looks, for
// roles that run ahead.
template <int NAP = 0>
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, const Abort& ab, int code) {
    constexpr uint32_t kLooks = NAP < 1000 ? 1u << 17 : 1u << 24;
    uint32_t ok, n = 0;
    while (!(ok = mbar_test(bar, parity)) && !*ab.flag) {
        if (++n == kLooks) *ab.flag = code;
        if (NAP) __nanosleep(NAP);
    }
    return __all_sync(0xffffffffu, ok);
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
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                 "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
          "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
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

// 2^((x - top) rf): the weight beside a maximum of top of what is relative to x (x at most top; both may be -inf).
__device__ __forceinline__ float lift_of(float x, float top, float rf) { return x == top ? 1.0f : exp2_f((x - top) * rf); }

// Items whose units several blocks had: blockIdx.x is the block that began it, a warp takes a row.  A kernel of its own: a
// block whose wait was given up would not be counted.
template <int DP>
__global__ void __launch_bounds__(128) attention_join(AttnArgs a) {
    pdl_begin();
    const int* m = (const int*)part_slot(a, kTileRows, DP, blockIdx.x, 1);
    if (!m[0]) return;
    const int row = blockIdx.y * 4 + (threadIdx.x >> 5);
    if (row >= m[2]) return;
    const int r = m[3] + row;
    join_row<kTileRows, DP>(a, blockIdx.x, m[5] - (int)blockIdx.x + 1, row, m[4] + r / a.group, m[1] * a.group + r % a.group);
}

// VEC: queries and outputs are 16-byte aligned.
template <int DP, bool VEC>
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
    uint64_t* fin_full = i_free + kItems;
    uint64_t* fin_free = fin_full + 1;
    uint64_t* sc_free = fin_free + 1;  // four each
    uint64_t* place_full = sc_free + 4;
    uint64_t* place_free = place_full + 4;
    uint32_t* tmem_slot = (uint32_t*)(place_free + 4);
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
            mbar_init(&p_full[i], kSoftThreads);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&sc_full[i], 32);
            mbar_init(&sc_free[i], kSoftWarps + 1);  // a lane of each warp that has read them, the issuer's too
            mbar_init(&place_full[i], 32);
            mbar_init(&place_free[i], 4);
        }
        for (int i = 0; i < kItems; ++i) {
            mbar_init(&i_full[i], 1);
            mbar_init(&i_free[i], kSoftWarps + 6);  // a lane of each softmax and sums warp, of the issuer and the guide
        }
        mbar_init(o_full, 2);  // the products' completion, and the issuer's arrival, which hands on what it has seen of P
        mbar_init(o_free, 128);
        mbar_init(fin_full, kSoftThreads);
        mbar_init(fin_free, 128);
        mbar_init(q_full, kSoftThreads);
        mbar_init(drain, 1);
        *gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kIssueWarp) {
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
        if (threads ? bar_any(id, threads, over) : __any_sync(0xffffffffu, over)) it.rows = it.n = 0;  // (what was read may be torn)
        return it;
    };

    if (!work) {
        // nothing to do but to free TMEM
    } else if (warp < kSoftWarps) {  // ---- softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
        constexpr int QD = DP / 2;  // this thread's values of a query
        const int half = warp >> 2, row = 32 * (warp & 3) + lane, pair = 1 + (warp & 3);  // barrier of a row's two warps
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        float* const maxima = (float*)(smem + C::MAXIMA) + row;
        uint32_t t = 0;  // tiles before the item's
#pragma unroll 1
        for (uint32_t i = 0;; ++i) {
            const TileItem it = item(i, pair, 64);
            if (!it.rows) break;
            const int r = it.first_row + row;
            const bool live = row < it.rows;
            float rf = 0.0f;
            if (it.n) {
                // the queries, as two f16 in TMEM, once the products that read the last item's are done
                const float* p = a.q + (int64_t)(it.row0 + (live ? r / a.group : 0)) * a.q_s1 +
                                 (int64_t)(it.head * a.group + (live ? r % a.group : 0)) * a.dim + QD * half;
                float* sums = (float*)(smem + C::SUMS) + row;
                uint32_t top = 0;
                float x[QD];
                if (VEC) {
#pragma unroll
                    for (int k = 0; k < QD / 4; ++k) {
                        const float4 v = live && QD * half + 4 * k < a.dim ? *(const float4*)(p + 4 * k) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        x[4 * k] = v.x, x[4 * k + 1] = v.y, x[4 * k + 2] = v.z, x[4 * k + 3] = v.w;
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < QD; ++k) x[k] = live && QD * half + k < a.dim ? p[k] : 0.0f;
                }
#pragma unroll
                for (int k = 0; k < QD; ++k) top = max(top, abs_bits(x[k]));
                sums[half * 128] = __uint_as_float(top);
                bar_named(pair, 64);
                top = max(top, __float_as_uint(sums[(half ^ 1) * 128]));
                bar_named(pair, 64);
                const float up = query_unit(top);
                if (t) {
                    warp_wait(&s_full[(t - 1) & 1], (t - 1) >> 1 & 1, ab, 43);
                    tc_fence_after();
                }
                const uint32_t at = tmem + lanes + C::Q_COL + QD / 2 * half;
#pragma unroll
                for (int c = 0; c < QD / 16; ++c) {
                    uint32_t h[8], lo[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) split2(x[16 * c + 2 * k] * up, x[16 * c + 2 * k + 1] * up, h[k], lo[k]);
                    tmem_st8(at + 8 * c, h);
                    tmem_st8(at + DP / 2 + 8 * c, lo);
                }
                tmem_st_done();
                rf = logit_unit(a.scale, up);
                if (half == 0) ((float*)(smem + C::FACTORS))[(i & 3) * 128 + row] = rf;
                tc_fence_before();
                mbar_arrive(q_full);
            }
            const int newest = live ? it.pos + r / a.group : -1, oldest = a.window && newest >= a.window ? newest - a.window + 1 : 0;
            const uint64_t rf2 = pair_of(rf, rf), top2 = pair_of(kTop, kTop);
            float m = -INFINITY, l = 0.0f;
#pragma unroll 1
            for (bool last = !it.n; !last; ++t) {
                const uint8_t* slot = smem + C::SCALES + (t & 3) * C::SLOT;
                const ulonglong2* ks = (const ulonglong2*)(slot + 64 * half * 4);
                const ulonglong2* vs = (const ulonglong2*)(slot + (kTileTokens + 64 * half) * 4);
                const uint32_t sc = tmem + lanes + C::S_COL + 128 * (t & 1) + 64 * half;
                bool on = warp_wait(&sc_full[t & 3], t >> 2 & 1, ab, 32);
                const int j0 = *(const int*)(slot + 2 * kTileTokens * 4 + 24);
                const uint4 ok = *(const uint4*)(slot + 2 * kTileTokens * 4);
                on &= warp_wait(&s_full[t & 1], t >> 1 & 1, ab, 33);
                tc_fence_after();
                uint64_t s[32];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t v[32];
                    tmem_ld32(sc + 32 * c, v);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const ulonglong2 kk = ks[8 * c + k];
                        s[16 * c + 2 * k] = mul2(pair_of(v[4 * k], v[4 * k + 1]), kk.x);
                        s[16 * c + 2 * k + 1] = mul2(pair_of(v[4 * k + 2], v[4 * k + 3]), kk.y);
                    }
                }
                // not all tokens seen by all rows
                if (j0 < it.all_first || j0 + kTileTokens - 1 > it.all_last || (ok.x & ok.y & ok.z & ok.w) != 0xffffffffu) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int at = j0 + 64 * half + 32 * c, lo = max(oldest - at, 0), hi = min(newest - at, 31);
                        const uint32_t bits = half ? (c ? ok.w : ok.z) : (c ? ok.y : ok.x);
                        const uint32_t seen = lo > hi ? 0u : bits & (0xffffffffu << lo) & (0xffffffffu >> (31 - hi));
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            float x, y;
                            unpair(s[16 * c + k], x, y);
                            s[16 * c + k] = pair_of(seen >> (2 * k) & 1 ? x : -INFINITY, seen >> (2 * k + 1) & 1 ? y : -INFINITY);
                        }
                    }
                }
                // the rows' maxima
                float x = -INFINITY, y = -INFINITY;
#pragma unroll
                for (int k = 0; k < 32; k += 2) {
                    float p, q;
                    unpair(s[k], p, q);
                    x = max3(x, p, q);
                    unpair(s[k + 1], p, q);
                    y = max3(y, p, q);
                }
                float* mine = maxima + (t & 1) * 256;
                mine[half * 128] = fmaxf(x, y);
                const float2 common = *(const float2*)(slot + 2 * kTileTokens * 4 + 16);
                const float unit = common.x;
                last = bar_any(pair, 64, common.y != 0.0f || !on);  // (both warps' answer is one, whatever was read after a wait was given up)
                const float top = fmaxf(mine[0], mine[128]);
                if (top > m) {
                    l *= m == -INFINITY ? 0.0f : exp2_f((m - top) * rf);
                    m = top;
                }
                const float ref = top == -INFINITY ? 0.0f : -top;  // (weights are relative to the tile's own maximum)
                const uint64_t ref2 = pair_of(ref, ref);
                const float lift = lift_of(top, m, rf);  // (of the tile's weights beside the row's)
                if (half == 0) ((float2*)(smem + C::REFS))[(t & 3) * 128 + row] = make_float2(m, copysignf(unit * lift, last ? -1.0f : 1.0f));
                uint64_t sum = 0;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t h[16], lo[16];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const ulonglong2 vv = vs[8 * c + k];
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            unpair(fma2(add2(s[16 * c + 2 * k + q], ref2), rf2, top2), x, y);
                            const uint64_t p = pair_of(exp2_f(x), exp2_f(y));
                            sum = add2(sum, p);
                            split_pair(mul2(p, q ? vv.y : vv.x), h[2 * k + q], lo[2 * k + q]);
                        }
                    }
                    tmem_st16(sc + 32 * c, h);
                    tmem_st16(sc + 32 * c + 16, lo);
                }
                unpair(sum, x, y);
                l = fmaf(x + y, lift, l);
                tmem_st_done();
                tc_fence_before();
                mbar_arrive(&p_full[t & 1]);
                if (lane == 0) mbar_arrive(&sc_free[t & 3]);
            }
            // the rows' sums, once the last item's have been read
            warp_wait<50>(fin_free, (i & 1) ^ 1, ab, 44);
            ((float*)(smem + C::STATS))[half * 128 + row] = l;
            mbar_arrive(fin_full);
        }
    } else if (warp < kLoadWarp) {  // ---- sums
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSumRegs));
        const int row = 32 * (warp & 3) + lane;
        const uint32_t oc = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + C::O_COL;
        uint32_t t = 0;
#pragma unroll 1
        for (uint32_t i = 0;; ++i) {
            const TileItem it = item(i, 0, 0);
            if (!it.rows) break;
            uint64_t o[DP / 2];
#pragma unroll
            for (int k = 0; k < DP / 2; ++k) o[k] = 0;
            float ref = -INFINITY, rf = 0.0f;
            // o is in units of `base`, a power of two that grows with the tiles' units and fades with the older weights, so that no sum
            // overflows; per = 1 / base.  (Not below kLeastBase, so that base / l is normal.)
            float base = kLeastBase, per = 1.0f / kLeastBase;
#pragma unroll 1
            for (bool last = !it.n; !last; ++t) {
                const bool on = warp_wait<100>(o_full, t & 1, ab, 31);
                tc_fence_after();
                rf = ((const float*)(smem + C::FACTORS))[(i & 3) * 128 + row];
                float2 mu = ((const float2*)(smem + C::REFS))[(t & 3) * 128 + row];
                last = __any_sync(0xffffffffu, signbit(mu.y) || !on);
                mu.y = fabsf(mu.y);
                if (__any_sync(0xffffffffu, mu.x > ref || mu.y > base)) {
                    const float fade = ref == mu.x ? 1.0f : exp2_f((ref - mu.x) * rf), held = base * fade;  // (from -inf: 0)
                    ref = mu.x;
                    base = unit_from(fmaxf(fmaxf(held, mu.y), kLeastBase)), per = one_by(base);
                    const uint64_t f = pair_of(held * per, held * per);
#pragma unroll
                    for (int k = 0; k < DP / 2; ++k) o[k] = mul2(o[k], f);
                }
                const uint64_t g = pair_of(mu.y * per, mu.y * per);
#pragma unroll
                for (int c = 0; c < DP / 16; ++c) {
                    uint32_t v[16];
                    tmem_ld16(oc + 16 * c, v);
                    if (c == DP / 16 - 1) {
                        tc_fence_before();
                        mbar_arrive(o_free);
                    }
#pragma unroll
                    for (int k = 0; k < 8; ++k) o[8 * c + k] = fma2(pair_of(v[2 * k], v[2 * k + 1]), g, o[8 * c + k]);
                }
            }
            warp_wait<100>(fin_full, i & 1, ab, 45);
            const float* stats = (const float*)(smem + C::STATS) + row;
            const float l = stats[0] + stats[128];
            mbar_arrive(fin_free);
            if (row < it.rows) {
                const int r = it.first_row + row;
                const float k = l == 0.0f ? 0.0f : base / l;
                const float top = top_of(ref, rf);
                float* dst;
                bool vec = VEC;
                if (it.whole) {
                    const int head = it.head * a.group + r % a.group;
                    const int64_t token = it.row0 + r / a.group;
                    dst = a.out + token * a.out_s1 + (int64_t)head * a.dim;
                    if (a.lse) a.lse[token * a.heads * a.group + head] = l == 0.0f ? -INFINITY : (top + log2f(l)) * kLn2;
                } else {
                    float* p = part_slot(a, kTileRows, DP, blockIdx.x, it.begins);
                    dst = p + 8 + 2 * kTileRows + row * DP, vec = true;
                    p[8 + 2 * row] = top, p[9 + 2 * row] = l;
                    if (row == 0 && it.begins) {
                        int* w = (int*)p;
                        w[1] = it.head, w[2] = it.rows, w[3] = it.first_row, w[4] = it.row0, w[5] = it.last_block, w[0] = 1;
                    }
                }
                const uint64_t kk = pair_of(k, k);
#pragma unroll
                for (int c = 0; c < DP / 4; ++c) {
                    float4 v;
                    unpair(mul2(o[2 * c], kk), v.x, v.y);
                    unpair(mul2(o[2 * c + 1], kk), v.z, v.w);
                    if (4 * c >= a.dim) continue;
                    if (vec) {
                        *(float4*)(dst + 4 * c) = v;
                    } else {
                        dst[4 * c] = v.x, dst[4 * c + 1] = v.y, dst[4 * c + 2] = v.z, dst[4 * c + 3] = v.w;
                    }
                }
            }
        }
    } else if (warp < kIssueWarp) {  // ---- loaders
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLoadRegs));
        constexpr int CH = DP / 16, PER = kTileTokens * CH / 128;  // pieces of 16 bytes of a row, and of a thread
        constexpr int STEP = 128 / CH;                             // rows between a thread's pieces
        // Eight lanes that store 16 bytes each have four pieces of two neighbouring rows, whose places in the swizzle differ by one:
        // no two have the same banks.
        const int tid = threadIdx.x - 32 * kLoadWarp, lw = warp - kLoadWarp;
        const int ch = CH == 8 ? (lane & 3) | (lane >> 1 & 4) : lane & 3;
        const int r0 = CH == 8 ? 4 * lw + (lane >> 2 & 1) + (lane >> 3 & 2) : 8 * lw + (lane >> 2);
        const uint32_t raw = smem_u32(smem + C::RAW) + tid * 16;
        const uint32_t piece = (uint32_t)(ch >> 2) * (kTileTokens * 128) + r0 * 128;
        uint8_t* at0 = smem + piece + ((2 * (ch & 3)) ^ (r0 & 7)) * 16;
        uint8_t* at1 = smem + piece + ((2 * (ch & 3) + 1) ^ (r0 & 7)) * 16;
        static_assert(STEP % 8 == 0, "a thread's rows have one place in the swizzle");
        if (a.stall) warp_wait(&k_empty[0], 0, ab, 34);  // a test of the bounded waits: nothing completes this phase
        // a thread's pieces of keys (0) or values (1) of the tile in stage st: as they came, to f16
        auto put = [&](int st, int which) {
            asm volatile("cp.async.wait_group 3;" ::: "memory");
            const uint8_t* from = smem + C::RAW + (2 * which + st) * C::RAW_TILE + tid * 16;
            const uint32_t tile = (2 * which + st) * C::TILE;
            uint4 v[PER];
#pragma unroll
            for (int k = 0; k < PER; ++k) v[k] = *(const uint4*)(from + k * 2048);
#pragma unroll
            for (int k = 0; k < PER; ++k) {
                *(uint4*)(at0 + tile + k * (STEP * 128)) =
                    make_uint4(f16_of_e4m3(v[k].x), f16_of_e4m3(v[k].x >> 16), f16_of_e4m3(v[k].y), f16_of_e4m3(v[k].y >> 16));
                *(uint4*)(at1 + tile + k * (STEP * 128)) =
                    make_uint4(f16_of_e4m3(v[k].z), f16_of_e4m3(v[k].z >> 16), f16_of_e4m3(v[k].w), f16_of_e4m3(v[k].w >> 16));
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        };
        const int64_t own = (int64_t)(r0 & 15) * a.dim + (16 * ch < a.dim ? 16 * ch : 0);
        uint32_t rows = 0;  // of the thread's pieces, those that exist
        auto fetch = [&](const uint8_t* from, const int64_t* places, int st, int which) {
            from += own;
            const uint32_t to = raw + (2 * which + st) * C::RAW_TILE;
            const uint8_t* p[PER];
#pragma unroll
            for (int k = 0; k < PER; ++k) p[k] = from + places[(STEP * k + r0) >> 4];
#pragma unroll
            for (int k = 0; k < PER; ++k) copy16(to + k * 2048, p[k], rows >> k & 1);
        };
        // Two tiles are on their way while one goes to f16, keys and values in turn; the tiles of the block's items follow one another
        // as the guide has them.
        uint32_t left = 0;  // tiles on their way
        bool more = true, have = false;
#pragma unroll 1
        for (uint32_t t = 0, x = 0, which = 0; more || left; which ^= 1) {  // t: the tile to put, x: to load
            uint64_t* full = k_full + 4 * which;  // (k_full, k_empty, v_full, v_empty)
            if (which == 0) have = left == 2 || !more;
            if (have) {
                warp_wait<200>(full + 2 + (t & 1), (t >> 1 & 1) ^ 1, ab, 34);
                put((int)(t & 1), (int)which);
                mbar_arrive(full + (t & 1));
                if (which) ++t, --left;
            }
            const int64_t* places = (const int64_t*)(smem + C::PLACES + (x & 3) * C::PLACE);
            if (which == 0 && more) {
                const bool found = warp_wait<200>(&place_full[x & 3], x >> 2 & 1, ab, 46) && places[0] >= 0;
                more = __all_sync(0xffffffffu, found);
                const uint4 ok = *(const uint4*)(places + 8);
                rows = 0xffu;
                if ((ok.x & ok.y & ok.z & ok.w) != 0xffffffffu) {
                    rows = 0;
#pragma unroll
                    for (int k = 0; k < PER; ++k) rows |= (((const uint32_t*)(places + 8))[(STEP * k + r0) >> 5] >> ((STEP * k + r0) & 31) & 1) << k;
                }
                if (16 * ch >= a.dim) rows = 0;
            }
            if (more) fetch(which ? a.v : a.k, places, (int)(x & 1), (int)which);
            asm volatile("cp.async.commit_group;" ::: "memory");
            if (which) {
                if (more) {
                    ++left;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&place_free[x & 3]);
                }
                ++x;
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
        if (warp == kIssueWarp) {  // ---- issuer
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
#pragma unroll 1
                    for (int h = 0; h < 2; ++h)
#pragma unroll 1
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
                for (bool last = false; ok && !last; ++t) {
                    ok = warp_wait(&sc_full[t & 3], t >> 2 & 1, ab, 49);
                    last = *(const float*)(smem + C::SCALES + (t & 3) * C::SLOT + 2 * kTileTokens * 4 + 20) != 0.0f;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sc_free[t & 3]);
                    if (ok && !last) logits(t + 1);
                    ok = ok && warp_wait(&v_full[t & 1], t >> 1 & 1, ab, 38);
                    ok = ok && warp_wait(&p_full[t & 1], t >> 1 & 1, ab, 39);
                    ok = ok && (t == 0 || warp_wait(o_free, (t - 1) & 1, ab, 40));
                    tc_fence_after();
                    if (ok && elect_one()) {
                        const uint32_t p = tmem + C::S_COL + 128 * (t & 1);
                        const uint64_t b = v0 + (uint64_t)((t & 1) * (C::TILE >> 4));
#pragma unroll 1
                        for (int h = 0; h < 2; ++h)
#pragma unroll 1
                            for (int s = 0; s < 8; ++s)
                                umma_ts(tmem + C::O_COL, p + 32 * (s >> 1) + 8 * (s & 1) + 16 * h, b + s * (2048 >> 4), io, h + s);
                        umma_commit(&v_empty[t & 1]);
                        umma_commit(o_full);
                        mbar_arrive(o_full);
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
        } else if (warp == kGuideWarp) {  // ---- guide: lane l has the tokens 4 l .. 4 l + 3 of a tile, of group l / 4
            // Tokens whose scales lie within 2^kNear share a unit, the least power of two above the largest, so that the weights' f16 halves
            // keep f32's bits beside the largest that a row sees.  Where a tile's differ by more it is taken in several rounds, of tokens
            // of like scales, largest first: tiles of the same places, of which other tokens are there.  (Scales of e^(s n), n normal, for s of
            // 0.3, 1, 2, 4 and 8: prompts 0.90, 1.25, 2.0, 3.4 and 5.9 ms; with one token of 2^-109 in every page 1.7.)
            uint32_t x = 0;  // the tile
#pragma unroll 1
            for (uint32_t i = 0;; ++i) {
                const TileItem it = item(i, 0, 0);
                const int32_t* table = a.table + (int64_t)it.seq * a.table_s1;
                int tok = it.first + 4 * lane, page = it.rows && it.n && (tok & ~15) < it.high ? table[tok >> a.page_log] : -1;
                bool on = it.rows != 0;
#pragma unroll 1
                for (int j = 0; j < (it.rows ? it.n : 1); ++j) {
                    const bool exists = (uint32_t)page < (uint32_t)a.pages;
                    const int64_t s = exists ? ((((int64_t)page * a.heads) + it.head) << a.page_log) + (tok & ((1 << a.page_log) - 1)) : (int64_t)(4 * (lane & 3));
                    uint32_t in = 0;  // which of the lane's four tokens exist
                    if (exists)
#pragma unroll
                        for (int q = 0; q < 4; ++q) in |= (uint32_t)(tok + q >= it.low && tok + q < it.high) << q;
                    const float4 ks = *(const float4*)(a.ks + s), vs = *(const float4*)(a.vs + s);
                    if (j + 1 < it.n) page = ((tok + kTileTokens) & ~15) < it.high ? table[(tok + kTileTokens) >> a.page_log] : -1;
                    const uint32_t all = __reduce_or_sync(0xffu << (lane & 24), in << 4 * (lane & 7));
                    float k[4] = {ks.x, ks.y, ks.z, ks.w}, v[4] = {vs.x, vs.y, vs.z, vs.w};
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        if (!(in >> q & 1)) k[q] = v[q] = 0.0f;
                        // (who sees a scale that is none is lost; none below zero is left, so that a round takes one token at least, the largest)
                        if (!(v[q] >= 0.0f && v[q] < kLargestScale) || !(fabsf(k[q]) < INFINITY)) k[q] = __uint_as_float(0x7FFFFFFFu), v[q] = 0.0f;
                    }
                    bool more;  // another round
                    do {
                        on = warp_wait<300>(&place_free[x & 3], (x >> 2 & 1) ^ 1, ab, 48) && on;
                        int64_t* places = (int64_t*)(smem + C::PLACES + (x & 3) * C::PLACE);
                        if ((lane & 3) == 0) places[lane >> 2] = it.rows ? s * a.dim : (int64_t)-1;  // (below zero: no more tiles)
                        if ((lane & 7) == 0) ((uint32_t*)(places + 8))[lane >> 3] = all;
                        mbar_arrive(&place_full[x & 3]);
                        if (!on) break;
                        uint32_t top = 0, take = 0;
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            if (in >> q & 1) top = max(top, abs_bits(v[q]));
                        top = __reduce_max_sync(0xffffffffu, top);
                        const float unit = unit_above(fmaxf(__uint_as_float(top), kLeastUnit)), per = one_by(unit);
                        float w[4];
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const bool like = in >> q & 1 && v[q] >= __uint_as_float(top) * kNear;
                            take |= (uint32_t)like << q;
                            w[q] = like ? v[q] * per : 0.0f;
                        }
                        in &= ~take;
                        more = __any_sync(0xffffffffu, in != 0);
                        warp_wait<300>(&sc_free[x & 3], (x >> 2 & 1) ^ 1, ab, 47);
                        uint8_t* slot = smem + C::SCALES + (x & 3) * C::SLOT;
                        ((float4*)slot)[lane] = make_float4(k[0], k[1], k[2], k[3]);
                        ((float4*)(slot + kTileTokens * 4))[lane] = make_float4(w[0], w[1], w[2], w[3]);
                        const uint32_t bits = __reduce_or_sync(0xffu << (lane & 24), take << 4 * (lane & 7));
                        if ((lane & 7) == 0) ((uint32_t*)(slot + 2 * kTileTokens * 4))[lane >> 3] = bits;
                        if (lane == 0)
                            *(float4*)(slot + 2 * kTileTokens * 4 + 16) =
                                make_float4(unit, j + 1 == it.n && !more ? 1.0f : 0.0f, __int_as_float(it.first + kTileTokens * j), 0.0f);
                        mbar_arrive(&sc_full[x & 3]);
                        ++x;
                    } while (more);
                    if (!on) break;
                    tok += kTileTokens;
                }
                if (!it.rows || *gave_up) break;
            }
        } else if (warp == kPlanWarp) {  // ---- planner
            for (uint32_t i = 0;; ++i) {
                TileItem p = {};
                const bool more = sh.more();
                if (more) {
                    const Item it = sh.item(a);
                    p.rows = it.rows, p.row0 = it.row0, p.first_row = it.first_row;
                    p.n = max(0, min(it.to, (it.high - it.base + kTileTokens - 1) / kTileTokens) - it.from);  // (the units behind the tokens hold none)
                    p.pos = it.pos, p.all_first = it.top_first, p.all_last = it.pos + it.first_row / a.group, p.head = it.head;
                    p.low = it.low, p.high = it.high, p.first = it.base + kTileTokens * it.from, p.seq = it.seq;
                    p.whole = it.from == 0 && it.to == it.units, p.begins = it.from == 0;
                    if (p.begins && !p.whole) p.last_block = sh.last_block(it);
                    sh.advance(a, it);
                }
                const bool ok = warp_wait<1000>(&i_free[i & (kItems - 1)], (i / kItems & 1) ^ 1, ab, 42);
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
    if (threadIdx.x == 0 && *gave_up) atomicCAS(a.status, 0, *gave_up);
    if (warp == kIssueWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
    }
}

template <int DP, bool VEC>
int run_tiles(const AttnArgs& a, cudaStream_t st) {
    static bool done[64];
    const cudaError_t e = allow_smem(attention_tiles<DP, VEC>, TileCfg<DP>::SMEM, done);
    if (e != cudaSuccess) return (int)e;
    const int rc = (int)launch_dep(attention_tiles<DP, VEC>, dim3((unsigned)a.blocks), dim3(kTileThreads), TileCfg<DP>::SMEM, st, a);
    if (rc) return rc;
    return (int)launch_dep(attention_join<DP>, dim3((unsigned)a.blocks, kTileRows / 4), dim3(128), 0, st, a);
}
template <int DP>
int run_tiles(const AttnArgs& a, cudaStream_t st) {
    return a.q_vec && a.out_vec ? run_tiles<DP, true>(a, st) : run_tiles<DP, false>(a, st);
}

}  // namespace
#endif
