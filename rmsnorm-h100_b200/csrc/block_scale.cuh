// block_scale.cuh -- what the 8-bit products and their quantisation share.
#pragma once

#include <type_traits>

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


__device__ __forceinline__ uint32_t octet_magnitude(const float2 (&v)[4]) { return magnitude(largest8(0.f, v)); }

// The largest of kLanes neighbouring lanes.
template <int kLanes>
__device__ __forceinline__ uint32_t largest_of(uint32_t m) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

// Eight values as they are loaded: 4 registers, 8 for fp32. Magnitudes of 16-bit values
// are compared as they are, two at a time: without the sign their bits order as unsigned integers,
// infinity above the numbers and NaN above it.
template <typename X>
struct Held {
  uint32_t w[4];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (uint32_t& x : w) x = 0;
  }
  __device__ __forceinline__ void load(const X* src) {  // whole, 16-byte aligned
    const uint4 u = RMSB_DBG_OK(src, 16, kDbgVecLoad) ? *reinterpret_cast<const uint4*>(src) : make_uint4(0, 0, 0, 0);
    w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
  }
  __device__ __forceinline__ void load(const X* src, int64_t n) {  // its first n values, one by one
    const uint16_t* bits = reinterpret_cast<const uint16_t*>(src);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      w[k] = (2 * k < n ? ld1(bits + 2 * k) : 0u) | (2 * k + 1 < n ? static_cast<uint32_t>(ld1(bits + 2 * k + 1)) << 16 : 0u);
  }
  __device__ __forceinline__ float2 pair(int k) const {
    if constexpr (std::is_same<X, __half>::value) return unpack_f16x2_pair(w[k]);
    else return unpack_bf16x2_pair(w[k]);
  }
  __device__ __forceinline__ static uint32_t widen(uint32_t m) {  // a magnitude's bits in fp32
    if constexpr (std::is_same<X, __half>::value)
      return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(m))));
    else return m << 16;
  }
};
template <>
struct Held<float> {
  float2 v[4];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (float2& x : v) x = make_float2(0.f, 0.f);
  }
  __device__ __forceinline__ void load(const float* src) { Pair8<float>::load(src, v); }
  __device__ __forceinline__ void load(const float* src, int64_t n) {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = make_float2(2 * k < n ? ld1(src + 2 * k) : 0.f, 2 * k + 1 < n ? ld1(src + 2 * k + 1) : 0.f);
  }
  __device__ __forceinline__ float2 pair(int k) const { return v[k]; }
};

__device__ __forceinline__ uint32_t larger2(uint32_t a, uint32_t b) {  // of both halves
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// The largest magnitude (fp32 bits) of each of kCount rows of kOctets octets a lane, over the
// kLanes lanes that share it.
template <typename X, int kLanes, int kCount, int kOctets = 1>
__device__ __forceinline__ void most_of(const Held<X> (&h)[kCount * kOctets], uint32_t (&most)[kCount]) {
  if constexpr (sizeof(X) == 4) {
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      uint32_t m = octet_magnitude(h[i * kOctets].v);
#pragma unroll
      for (int o = 1; o < kOctets; ++o) m = max(m, octet_magnitude(h[i * kOctets + o].v));
      most[i] = largest_of<kLanes>(m);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kCount; i += 2) {
      uint32_t m[2] = {0, 0};
#pragma unroll
      for (int k = 0; k < 2 && i + k < kCount; ++k)
#pragma unroll
        for (int o = 0; o < kOctets; ++o) {
          const uint32_t(&w)[4] = h[(i + k) * kOctets + o].w;
          const uint32_t one = larger2(larger2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu), larger2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
          m[k] = o ? larger2(m[k], one) : one;
        }
      // row i's in the low half, the next one's in the high half
      uint32_t both = larger2(__byte_perm(m[0], m[1], 0x5410), __byte_perm(m[0], m[1], 0x7632));
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) both = larger2(both, __shfl_xor_sync(0xffffffffu, both, o));
      most[i] = Held<X>::widen(both & 0xffffu);
      if (i + 1 < kCount) most[i + 1] = Held<X>::widen(both >> 16);
    }
  }
}

}  // namespace rmsb200
