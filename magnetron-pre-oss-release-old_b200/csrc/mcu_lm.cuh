// Device helpers of the language-model row kernels (norm, e4m3 quantiser and product, log probabilities).
#ifndef MCU_LM_CUH
#define MCU_LM_CUH
#include <cstdint>

namespace mcu {

constexpr float kE4m3Max = 448.0f;
// The smallest largest magnitude a scale is formed from, 2^-100: the scale and its reciprocal stay
// normal f32 values, so a group of zeros (or of subnormals) divides cleanly.
constexpr float kE4m3Tiny = 7.8886090522101181e-31f;

// Four values as e4m3 bytes, a in the lowest; rounded to nearest even, saturating, NaN kept.
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return (uint32_t)lo | ((uint32_t)hi << 16);
}

// |v| as an integer whose order is the magnitude's, NaN above infinity: a maximum over these keeps NaN.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// A group's scale s, a / 448 (a its largest magnitude, at least kE4m3Tiny) by a multiplication, from the bits of that
// magnitude, and two factors around 1 / s.  With u = 2^-24, c = 1 / 448 as f32 holds it is (1 / 448)(1 + 0.75 u), so that
// s = a c (1 + d1) = (a / 448)(1 + d), |d| <= 1.76 u.  f = (448 / a)(1 + d2), hence 1 / s lies within f (1 +- 2.8 u), and
// low and high = f (1 -+ 4 u)(1 + d3) lie outside that (d1, d2, d3 are single roundings, at most u).
struct E4m3Group {
    float scale, low, high;
};
__device__ __forceinline__ E4m3Group e4m3_group(uint32_t amax_bits) {
    const float a = __uint_as_float(amax_bits), m = a < kE4m3Tiny ? kE4m3Tiny : a, f = __fdiv_rn(kE4m3Max, m);
    return E4m3Group{__fmul_rn(m, 1.0f / kE4m3Max), __fmul_rn(f, 1.0f - 0x1p-22f), __fmul_rn(f, 1.0f + 0x1p-22f)};
}
__device__ __forceinline__ uint32_t e4m3_divide(float scale, float a, float b, float c, float d) {
    return e4m3x4(__fdiv_rn(a, scale), __fdiv_rn(b, scale), __fdiv_rn(c, scale), __fdiv_rn(d, scale));
}
// Four values as bytes: each quotient v / s rounded to f32, then to e4m3.  Rounding keeps order, so where v low and
// v high give the same byte the quotient gives it too; else (5 values of 10^6, those next to a tie) *open gets a bit,
// and the quotients have to be formed.  On the device an 8192 x 4096 weight turned, in blocks, takes 30.4 us so, 37.9
// when every value is divided, and 27.9 by one factor alone, which moved one value of 3 * 10^6 to its other neighbour.
__device__ __forceinline__ uint32_t e4m3_try(const E4m3Group& g, float a, float b, float c, float d, uint32_t* open) {
    const uint32_t q = e4m3x4(a * g.low, b * g.low, c * g.low, d * g.low);
    *open |= q ^ e4m3x4(a * g.high, b * g.high, c * g.high, d * g.high);
    return q;
}
__device__ __forceinline__ uint32_t e4m3_quotients(const E4m3Group& g, float a, float b, float c, float d) {
    uint32_t open = 0;
    const uint32_t q = e4m3_try(g, a, b, c, d, &open);
    return open ? e4m3_divide(g.scale, a, b, c, d) : q;
}

__device__ __forceinline__ float warp_sum_f(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

}  // namespace mcu
#endif
