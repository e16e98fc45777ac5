// block_scale.cuh -- what the 8-bit products and their quantisation share.
#pragma once

#include "fused_common.cuh"

namespace rmsb200 {

constexpr int kBlock = RMSNORM_B200_BLOCK;  // columns of a scale's group, rows and columns of its block

// The smallest power of two that brings a magnitude (its bits) to 448 = 1.75 * 2^8 or below, at
// least 2^-126; infinity and NaN stay. A power of two makes x / scale exact, so that a value has
// one nearest e4m3 number whatever the order of operations, and value * scale exact in every
// floating type; e4m3 loses nothing by it but up to one of its 15 octaves.
__device__ __forceinline__ uint32_t power_scale(uint32_t largest) {
  const uint32_t e = largest >> 23, above = (largest & 0x7fffffu) > 0x600000u ? 1u : 0u;
  if (e == 255) return largest;
  return (e + above <= 9 ? 1u : e + above - 8) << 23;
}

// 1 / scale: exact for a power of two from 2^-126 to 2^120, 0 for infinity, NaN for NaN.
__device__ __forceinline__ float power_inverse(uint32_t scale) {
  if (scale >= 0x7f800000u) return scale > 0x7f800000u ? __uint_as_float(scale) : 0.f;
  return __uint_as_float((254u << 23) - scale);
}

}  // namespace rmsb200
