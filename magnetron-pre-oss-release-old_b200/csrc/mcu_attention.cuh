// Pieces that the attention kernels share: how blocks share the work, what an item is, and where its output goes.
#ifndef MCU_ATTENTION_CUH
#define MCU_ATTENTION_CUH
#include <cuda_runtime.h>
#include <cstdint>
#include "mcu_kernels.h"
#include "mcu_launch.cuh"
#include "mcu_lm.cuh"

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;
constexpr float kNone = -3.0e38f;               // the maximum of no logits: finite, so that differences of it stay numbers
constexpr float kTop = 15.0f;                   // probabilities are formed as 2^kTop p: their f16 halves keep 22 bits down to 2^-18
// Weights p s (probability times the value's scale) are formed in units of a power of two above the largest of a row's, so that
// their f16 halves hold them to 2^-40 of that: of what the row itself sees, whatever else lies beside it, and however small the
// probabilities are.
constexpr float kLeastUnit = 0x1p-110f;         // a row's unit before any weight was seen (the least scale is 2^-109)
constexpr float kLargestScale = 0x1p126f;       // a scale that is no number or not finite does not set the unit
constexpr int kUnitTokens = 128;                // tokens of a unit of work

struct AttnArgs {
    float *out, *lse;
    const float* q;
    const uint8_t *k, *v;
    const float *ks, *vs;
    const int32_t *table, *start, *length;
    int64_t table_s1, q_s1, out_s1;
    float* parts;  // two slots a block, of part_floats() floats
    int* status;
    uint32_t* joins;  // attention_few's counters, one a block: parts of the item that the block begins
    int seqs, rows, max_new, heads, group, dim, pages, page_log, window;
    int longest;             // tokens that a sequence's table has room for
    int least, most;         // the rows of a kv head (new tokens x group) of the sequences that this launch takes
    int blocks, q_vec, out_vec, stall;
    float scale;
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ float4 four_of(const float* p, int vec) {
    if (vec) return *(const float4*)p;
    return make_float4(p[0], p[1], p[2], p[3]);
}
__device__ __forceinline__ float exp2_f(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ void store_row(const AttnArgs& a, int64_t row, int head, int d, float4 v) {
    float* p = a.out + row * a.out_s1 + (int64_t)head * a.dim + d;
    if (a.out_vec) {
        *(float4*)p = v;
    } else {
        p[0] = v.x, p[1] = v.y, p[2] = v.z, p[3] = v.w;
    }
}
// The logarithm (base 2) of the probabilities' unit where the highest logit is m, in units of rf; kNone for no logits.
__device__ __forceinline__ float top_of(float m, float rf) { return m == -INFINITY ? kNone : fmaf(m, rf, -kTop); }
// Two e4m3 bytes (the low ones of x) as two f16, exactly.
__device__ __forceinline__ uint32_t f16_of_e4m3(uint32_t x) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)x));
    return r;
}
// a and b as f16 pairs (a low): high = the nearest f16, low = the nearest f16 of what is left, 22 bits together.
__device__ __forceinline__ void split2(float a, float b, uint32_t& high, uint32_t& low) {
    asm("{\n\t.reg .b16 x, y;\n\t.reg .f32 u, v;\n\t"
        "cvt.rn.f16x2.f32 %0, %3, %2;\n\t"
        "mov.b32 {x, y}, %0;\n\t"
        "cvt.f32.f16 u, x;\n\t"
        "cvt.f32.f16 v, y;\n\t"
        "sub.f32 u, %2, u;\n\t"
        "sub.f32 v, %3, v;\n\t"
        "cvt.rn.f16x2.f32 %1, v, u;\n\t}"
        : "=&r"(high), "=r"(low)
        : "f"(a), "f"(b));
}
// The power of two that takes a query row of largest magnitude `top` (its bits) to 2^13 .. 2^14, where both halves of a
// value have their bits, or as near to it as 2^126 does (rows of zeros and of the smallest values); 1 for a row with a NaN or infinity.
__device__ __forceinline__ float query_unit(uint32_t top) {
    const int e = (int)(top >> 23);
    return e == 255 ? 1.0f : __uint_as_float((uint32_t)min(253, 127 + 127 + 13 - e) << 23);
}
// The least power of two above v (v finite, positive, below 2^126).
__device__ __forceinline__ float unit_above(float v) { return __uint_as_float((__float_as_uint(v) & 0x7F800000u) + 0x00800000u); }

// The least power of two not below v (v positive and normal, at most 2^126), and 1 / v of such a power.
__device__ __forceinline__ float unit_from(float v) { return __uint_as_float((__float_as_uint(v) + 0x007FFFFFu) & 0x7F800000u); }
__device__ __forceinline__ float one_by(float v) { return __uint_as_float(0x7F000000u - __float_as_uint(v)); }

// What takes a logit of queries times `up` to powers of two: finite, and above zero, so that -inf times it is -inf.
__device__ __forceinline__ float logit_unit(float scale, float up) { return fminf(fmaxf(scale * one_by(up) * kLog2e, 0x1p-126f), 3.402823466e38f); }

// Where a piece of 16 bytes of a staged row of keys or values lies within its row, so that the lanes that read
// together find other banks.
template <int DP>
__device__ __forceinline__ int key_chunk(int ch, int row) {
    return DP == 128 ? ch ^ 4 * (row & 1) : ch;
}
template <int DP>
__device__ __forceinline__ int value_chunk(int ch, int row) {
    return DP == 128 ? ch ^ (row & 6) : ch ^ (row >> 1 & 3);
}
// What the place of a piece of values changes by, in bytes, from row r0 to row r0 + i 512 / DP (r0 below 512 / DP).
template <int DP>
__device__ __forceinline__ constexpr uint32_t value_turn(int i) {
    return DP == 128 ? 16 * (4 * i & 6) : 0;
}

// One item: up to MAX rows (new token, query head of the group) of a sequence and kv head, and this block's part of the
// tokens that they see.  Row r of the item is row first_row + r of the sequence's rows, of token (first_row + r) / group.
struct Item {
    int seq, head, rows, first_row;
    int row0;             // the sequence's first row of q and out
    int pos;              // position of the sequence's first new token (negative where it is not in the cache)
    int low, high, base;  // tokens that any row sees; base = low rounded down to whole groups of 16
    int top_first;        // the first token that all rows see
    int units, from, to;  // units of 128 tokens from base, and this block's
};

// Tokens that the rows [first_row, first_row + rows) of a sequence see together.
struct Seq {
    int row0, n, take, length;  // take: rows of q that are taken (at most max_new)
    __device__ Seq() {}
    __device__ Seq(const AttnArgs& a, int s) {
        row0 = min(max(a.start[s], 0), a.rows);
        const int end = min(max(a.start[s + 1], row0), a.rows);
        n = end - row0;
        take = min(n, a.max_new);
        length = min(max(a.length[s], 0), a.longest);
        const int64_t rows = (int64_t)take * a.group;
        if (rows < a.least || rows > a.most) take = 0;
    }
};
__device__ __forceinline__ int first_seen(const AttnArgs& a, int pos) { return a.window && pos >= a.window ? pos - a.window + 1 : 0; }

template <int MAX>
__device__ __forceinline__ int64_t tiles_of(const AttnArgs& a, const Seq& q) {
    return ((int64_t)q.take * a.group + MAX - 1) / MAX;
}
// Tokens and units of tile t of a sequence: at least one unit, so that rows that see nothing are written.  Tiles of many rows
// count kItemUnits more, for what an item costs besides its tokens (its queries, its output, the way from one to the next): four
// prompts of up to 4100 tokens took 1090, 967, 895, 913 and 945 us with 0, 2, 4, 6 and 8 more, with a window of 1000 723, 657, 638,
// 642 and 640, three chunks of up to 300 over 20000 204, 198, 196, 199 and 201; 100 prompts of up to 100 tokens 166 to 167 with each.
constexpr int kItemUnits = 4;
template <int MAX>
__host__ __device__ constexpr int extra_units() {
    return MAX > 16 ? kItemUnits : 0;
}
template <int MAX>
__device__ __forceinline__ int span_of(const AttnArgs& a, const Seq& q, int64_t t, int& low, int& high) {
    const int tok0 = (int)(t * MAX / a.group), tok1 = (int)(min(t * MAX + MAX, (int64_t)q.take * a.group) - 1) / a.group;
    const int p0 = q.length - q.n + tok0, p1 = q.length - q.n + tok1;
    low = first_seen(a, p0), high = p1 + 1;
    if (high <= low) low = high = 0;
    return max(1, (high - (low & ~15) + kUnitTokens - 1) / kUnitTokens + extra_units<MAX>());
}

// A slot of a block's part of an item: 8 ints (attention_tiles alone uses them: 1 if it begins an item that ends elsewhere, the item's
// head, rows, first row, row0, last block), then maximum and sum of each row, then its rows of output.
__host__ __device__ constexpr int64_t part_floats(int max, int dp) { return 8 + 2 * max + (int64_t)max * dp; }
__device__ __forceinline__ float* part_slot(const AttnArgs& a, int max, int dp, int64_t block, int which) {
    return a.parts + (2 * block + which) * part_floats(max, dp);
}

// a / b for a from 0 to 2^53, b above 0: in 32 bits where both fit, else the f64 quotient, which is off by one at most.  (The
// compiler's 64-bit division is a long way round.)
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    if (((a | b) >> 32) == 0) return (uint32_t)a / (uint32_t)b;
    int64_t q = (int64_t)((double)a / (double)b);
    const int64_t r = a - q * b;
    return r < 0 ? q - 1 : r >= b ? q + 1 : q;
}

// A share's end moves to the beginning or end of its item where that is no further than so many units, the item's middle and half
// a share: a block that begins an item pays for it what some units of tokens cost (four sequences of up to 2000 tokens 18.2 -> 13.6
// us, eight of 64 values a head 16.7 -> 13.4; up to 3 units 15.4 and 14.1, and without the bound of half a share one sequence of 500
// tokens took 11.5 us, 10.8 with it).  Few rows; with many, an item's own units (kItemUnits) stand for that.
constexpr int kSnapUnits = 2;

// A block's share of all units, in the order sequence, kv head, tile, tokens: equal shares, so that ragged lengths load
// the GPU evenly whatever the lengths are, which only the device knows.  An item that a share's end cuts is joined from its
// parts afterwards.  THREADS threads of the block look for its first item together; each of them, or some, then goes on alone.
template <int MAX, int DP, int THREADS>
struct Share {
    static constexpr bool BY_WARP = MAX > 16;  // a sequence has many tiles: the lanes of a warp share them
    static constexpr int WARPS = THREADS / 32, SMEM = 32 * 8 + 48 + 16;
    int64_t total, at, left, tile;
    int blocks, seq, head, off, reach;
    Seq here;  // the sequence at hand

    // Units of one kv head of a sequence.
    __device__ static int64_t seq_units(const AttnArgs& a, const Seq& q) {
        const int64_t n = tiles_of<MAX>(a, q);
        int64_t u = 0;
        int lo, hi;
        if constexpr (!BY_WARP) {
            u = n ? span_of<MAX>(a, q, 0, lo, hi) : 0;
        } else {
            for (int64_t t = threadIdx.x & 31; t < n; t += 32) u += span_of<MAX>(a, q, t, lo, hi);
#pragma unroll
            for (int o = 16; o; o >>= 1) u += __shfl_xor_sync(0xffffffffu, u, o);
        }
        return u;
    }
    // The first unit of block b, before it is moved to an item's beginning or end.
    __device__ int64_t begin_of(int b) const { return quotient(total * b, blocks); }
    // Finds the block's first item; false when the block has no work.  sh: SMEM bytes of shared memory.
    __device__ bool find(const AttnArgs& a, int64_t* sh) {
        int64_t* found = sh + 32;
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        if (MAX > 16 && threadIdx.x == 0) *(int*)slot(a, 1) = 0;
        // each thread (or warp) has a run of sequences
        const int workers = BY_WARP ? WARPS : THREADS, me = BY_WARP ? warp : threadIdx.x;
        const int run = (a.seqs + workers - 1) / workers, s0 = min(me * run, a.seqs), s1 = min(s0 + run, a.seqs);
        int64_t mine = 0;
#pragma unroll 1
        for (int s = s0; s < s1; ++s) mine += seq_units(a, Seq(a, s)) * a.heads;
        int64_t inc = mine;
        if (!BY_WARP) {
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t t = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += t;
            }
        }
        if (lane == 31) sh[warp] = inc;
        __syncthreads();
        int64_t before = 0;
        total = lane < WARPS ? sh[lane] : 0;
        before = lane < warp ? total : 0;
#pragma unroll
        for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o), before += __shfl_xor_sync(0xffffffffu, before, o);
        before += inc - mine;
        blocks = (int)min((int64_t)gridDim.x, total);  // each has a unit at least, so that an item's parts lie in consecutive blocks
        if ((int)blockIdx.x >= blocks) return false;
        at = begin_of(blockIdx.x);
        reach = BY_WARP ? 0 : (int)min((int64_t)kSnapUnits, quotient(total, blocks) / 2);
        left = begin_of(blockIdx.x + 1) - at;
        if (!BY_WARP) {
            const int64_t end = at + left;
            if (end >= before && end < before + mine) {
                int64_t x = end - before, u = 0;
#pragma unroll 1
                for (int s = s0; s < s1; ++s) {
                    u = seq_units(a, Seq(a, s)) * a.heads;
                    if (x < u) break;
                    x -= u;
                }
                found[6] = moved(x, (int)quotient(u, a.heads)) - x;
            }
            if (end == total && threadIdx.x == 0) found[6] = 0;
        }
        if (at >= before && at < before + mine) {
            int64_t x = at - before, u = 0;
            int s = s0;
            Seq q;
#pragma unroll 1
            for (; s < s1; ++s) {
                q = Seq(a, s);
                u = seq_units(a, q);
                if (x < u * a.heads) break;
                x -= u * a.heads;
            }
            if (!BY_WARP || lane == 0) {
                found[0] = s, found[1] = x, found[2] = u;
                *(int4*)(found + 4) = make_int4(q.row0, q.n, q.take, q.length);
            }
        }
        __syncthreads();
        seq = (int)found[0];
        const int4 h = *(const int4*)(found + 4);
        here.row0 = h.x, here.n = h.y, here.take = h.z, here.length = h.w;
        const int64_t x = found[1], per = found[2];
        head = (int)quotient(x, per);
        int64_t rest = x - head * per;
        tile = 0;
        if (!BY_WARP) {
            const int64_t to = moved(x, (int)per) - x;
            at += to, left += found[6] - to, rest += to;
            if (left <= 0) return false;
            if (rest == per) rest = 0, next_head(a);
        }
        if (BY_WARP) {  // (each warp for itself)
            const int64_t n = tiles_of<MAX>(a, here);
#pragma unroll 1
            for (;; tile += 32) {
                int lo, hi;
                const int64_t u = tile + lane < n ? span_of<MAX>(a, here, tile + lane, lo, hi) : 0;
                inc = u;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int64_t t = __shfl_up_sync(0xffffffffu, inc, o);
                    if (lane >= o) inc += t;
                }
                const uint32_t past = __ballot_sync(0xffffffffu, inc > rest);
                if (past) {
                    const int i = __ffs((int)past) - 1;
                    tile += i;
                    rest -= __shfl_sync(0xffffffffu, inc - u, i);
                    break;
                }
                rest -= __shfl_sync(0xffffffffu, inc, 31);
                if (tile + 32 >= n) break;  // (not reached: the sequence's units hold the unit looked for)
            }
        }
        off = (int)rest;
        __syncthreads();
        return true;
    }
    // Where unit x of a sequence, `units` to a head, is moved to.
    __device__ int64_t moved(int64_t x, int units) const {
        const int64_t first = quotient(x, units) * units;
        const int r = (int)(x - first), t = min(reach, units / 2);
        return r <= t ? first : units - r <= t ? first + units : x;
    }
    __device__ void next_head(const AttnArgs& a) {
        if (++head < a.heads) return;
        head = 0;
        while (++seq < a.seqs) {
            here = Seq(a, seq);
            if (here.take) return;
        }
        left = 0;  // (not reached: the shares add up to all units)
    }
    __device__ bool more() const { return left > 0; }
    __device__ Item item(const AttnArgs& a) const {
        const Seq& q = here;
        Item it;
        it.seq = seq, it.head = head, it.row0 = q.row0;
        it.first_row = (int)(tile * MAX);
        it.rows = (int)min((int64_t)MAX, (int64_t)q.take * a.group - it.first_row);
        it.pos = q.length - q.n;
        it.units = span_of<MAX>(a, q, tile, it.low, it.high);
        it.base = it.low & ~15;
        it.top_first = first_seen(a, it.pos + (it.first_row + it.rows - 1) / a.group);
        it.from = off;
        it.to = (int)min((int64_t)it.units, off + left);
        return it;
    }
    __device__ void advance(const AttnArgs& a, const Item& it) {
        at += it.to - it.from, left -= it.to - it.from, off = 0;
        if (left <= 0) return;
        if (MAX > 16) {
            ++tile;
            if (tile < tiles_of<MAX>(a, here)) return;
        }
        tile = 0;
        next_head(a);
    }
    // The blocks that hold the first and the last unit of the item at hand.
    __device__ int first_block(const Item& it) const {
        return it.from ? block_of(at - it.from + min(reach, it.units / 2)) : (int)blockIdx.x;
    }
    __device__ int last_block(const Item& it) const {
        const int t = min(reach, it.units / 2);
        return block_of(at - it.from + max(it.units - 1 - t, t));
    }
    // The last block whose share, before it is moved, begins at or before unit x.
    __device__ int block_of(int64_t x) const {
        int b = (int)quotient((x + 1) * blocks, total);
        while (begin_of(b) > x) --b;
        while (begin_of(b + 1) <= x) ++b;
        return b;
    }
    __device__ static float* slot(const AttnArgs& a, int which) { return part_slot(a, MAX, DP, blockIdx.x, which); }
};

// Row `row` of an item whose units the blocks [first, first + parts) had; a warp.  The parts' weights are their sums times
// 2^(top - the highest top); parts are added in the blocks' order.
template <int MAX, int DP>
__device__ __forceinline__ void join_row(const AttnArgs& a, int first, int parts, int row, int64_t to, int head) {
    const int lane = threadIdx.x & 31;
    auto stats = [&](int p) {
        return p < parts ? __ldcg((const float2*)(part_slot(a, MAX, DP, first + p, p == 0) + 8 + 2 * row)) : make_float2(kNone, 0.0f);
    };
    auto values = [&](int p) {
        return p < parts && 4 * lane < DP ? __ldcg((const float4*)(part_slot(a, MAX, DP, first + p, p == 0) + 8 + 2 * MAX + row * DP + 4 * lane))
                                          : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    };
    const float2 mine = stats(lane);
    float4 t[4];  // the next parts' values, under way
#pragma unroll
    for (int k = 0; k < 4; ++k) t[k] = values(k);
    float top = mine.x, total = 0.0f;
    for (int p = lane + 32; p < parts; p += 32) top = fmaxf(top, stats(p).x);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    // a power of two that keeps the weights' sum, at most 2^kTop a token, at 1 or below: no sum of values overflows
    const float less = one_by(unit_from((float)a.longest)) * 0x1p-15f;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int p0 = 0; p0 < parts; p0 += 32) {
        const float2 s = p0 ? stats(p0 + lane) : mine;
        const float w = p0 + lane < parts ? s.y * less * exp2_f(s.x - top) : 0.0f;
        const int n = min(32, parts - p0);
#pragma unroll 1
        for (int i = 0; i < n; i += 4) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float f = __shfl_sync(0xffffffffu, w, i + k);  // (zero past the parts)
                total += f;
                v.x = fmaf(f, t[k].x, v.x), v.y = fmaf(f, t[k].y, v.y), v.z = fmaf(f, t[k].z, v.z), v.w = fmaf(f, t[k].w, v.w);
                t[k] = values(p0 + i + 4 + k);
            }
        }
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    if (4 * lane < a.dim) store_row(a, to, head, 4 * lane, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
    total /= less;
    if (lane == 0 && a.lse) a.lse[to * a.heads * a.group + head] = total == 0.0f ? -INFINITY : (top + log2f(total)) * kLn2;
}

}  // namespace
#endif
