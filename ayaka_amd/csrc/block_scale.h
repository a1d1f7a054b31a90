// The scales of a block-scaled 8-bit cache (codec "fp8_e4m3_block"): float32
// [num_blocks, num_kv_heads, 2], a key scale and a value scale for every block and key/value
// head. A scale is a power of two 2^e, kLeast <= e <= kMost, or 0 for a block that holds nothing
// but zeros (its codes then decode to zeros at any scale).
//
// Powers of two, because e4m3 is a floating format: its relative precision does not depend on
// the scale, so a finer scale would gain nothing, while a block whose scale grows by 2^k
// re-encodes its tokens by lowering their exponents: exact for every code that stays normal.
// The range of e keeps every ratio of two scales (2^120), and every sum of weights in units of one,
// inside fp32; what a weight in units of the largest scale loses, the attention kernels' sums take
// from exponentials of their own (PositionScale).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace ayk {

constexpr int kScaleLeast = -40;
constexpr int kScaleMost = 80;

#define AYK_SCALE_HD __host__ __device__ __forceinline__

AYK_SCALE_HD uint32_t float_bits(float f) { return __builtin_bit_cast(uint32_t, f); }
AYK_SCALE_HD float bits_float(uint32_t u) { return __builtin_bit_cast(float, u); }

// 2^e for -126 <= e <= 127.
AYK_SCALE_HD float power_of_two(int e) { return bits_float((uint32_t)(e + 127) << 23); }

// The exponent of a scale as stored, clamped to the range (whatever the memory holds: a value
// that is no power of two counts as the one below it, infinities and NaN as the largest).
AYK_SCALE_HD int scale_exponent(float s) {
  const int e = (int)((float_bits(s) >> 23) & 0xffu) - 127;
  return e < kScaleLeast ? kScaleLeast : e > kScaleMost ? kScaleMost : e;
}

// A scale as stored, made one the codec allows: 0 for anything not above 0.
AYK_SCALE_HD float canonical_scale(float s) {
  const uint32_t u = float_bits(s);
  return (u - 1u) < 0x7fffffffu ? power_of_two(scale_exponent(s)) : 0.f;  // 0 < u < 2^31: sign clear, not +0
}

// The least scale that keeps magnitudes up to `amax` (finite) within e4m3's 448 = 1.75 * 2^8;
// 0 for 0. Above 448 * 2^kScaleMost the codes saturate.
AYK_SCALE_HD float scale_for(float amax) {
  const uint32_t u = float_bits(amax);
  if (u == 0) return 0.f;
  const int e = (int)(u >> 23) - 127 - ((u & 0x7fffffu) <= 0x600000u ? 8 : 7);
  return power_of_two(e < kScaleLeast ? kScaleLeast : e > kScaleMost ? kScaleMost : e);
}

}  // namespace ayk
