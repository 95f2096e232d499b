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

// A group's scale amax / 448 and the factor 448 / amax of its values, from the bits of its largest
// magnitude.  A value is rounded twice in f32 (the factor, the product) before e4m3 rounds it, which moves
// about one in 10^7, those within 2^-23 of a tie, to the neighbour that lies as near.  The corrected division
// (two fused multiply-adds a value) cost 4 to 15 % of the kernels and still rounds once in f32.
struct E4m3Group {
    float scale, factor;
};
__device__ __forceinline__ E4m3Group e4m3_group(uint32_t amax_bits) {
    const float a = __uint_as_float(amax_bits), m = a < kE4m3Tiny ? kE4m3Tiny : a;
    return E4m3Group{__fdiv_rn(m, kE4m3Max), __fdiv_rn(kE4m3Max, m)};
}

__device__ __forceinline__ float warp_sum_f(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

}  // namespace mcu
#endif
