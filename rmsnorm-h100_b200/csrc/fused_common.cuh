// fused_common.cuh -- the mathematics shared by the fused row operators: the dropout mask,
// and 8-bit values with scales.
#pragma once

#include <cuda_fp8.h>

#include "device_common.cuh"

namespace rmsb200 {

// ---------------------------------------------------------------------------------------
// Dropout mask: Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy
// as 1, 2, 3; SC 2011), one call per four columns. The counter holds the column, the row and
// the caller's offset, so a mask needs no memory, the backward draws it again, and a rank
// that holds some rows of a tensor draws those rows of the whole tensor's mask.
// The round keys depend on the seed alone: the host expands them, and the kernels read them
// as constants (two multiplications and two three-way xors a round).
// ---------------------------------------------------------------------------------------
struct DropParams {
  uint32_t key[20];       // round r: key[2r], key[2r + 1]
  uint64_t offset;
  const int64_t* step;    // nullable: added to the offset when the kernel runs
  int64_t row0;           // row_offset
  uint32_t least;         // a word below it drops its element: floor(p * 2^32)
  float scale;            // 1 / (1 - p)
};

constexpr uint32_t kPhiloxM0 = 0xD2511F53u, kPhiloxM1 = 0xCD9E8D57u;
constexpr uint32_t kPhiloxW0 = 0x9E3779B9u, kPhiloxW1 = 0xBB67AE85u;

inline void expand_drop(const rmsnorm_b200_dropout& d, DropParams* p) {
  uint32_t k0 = static_cast<uint32_t>(d.seed), k1 = static_cast<uint32_t>(d.seed >> 32);
  for (int r = 0; r < 10; ++r) {
    p->key[2 * r] = k0;
    p->key[2 * r + 1] = k1;
    k0 += kPhiloxW0;
    k1 += kPhiloxW1;
  }
  p->offset = d.offset;
  p->step = d.step;
  p->row0 = d.row_offset;
  p->least = static_cast<uint32_t>(d.p * 4294967296.0);
  p->scale = static_cast<float>(1.0 / (1.0 - d.p));
}

inline bool valid_drop(const rmsnorm_b200_dropout& d, int64_t rows) {
  return d.p >= 0.0 && d.p < 1.0 && d.row_offset >= 0 && d.row_offset <= (int64_t{1} << 32) - rows;
}

// The offset of this execution (after the kernel's pdl_wait).
__device__ __forceinline__ uint64_t drop_offset(const DropParams& d) {
  return d.offset + (d.step ? static_cast<uint64_t>(ld1(d.step)) : 0ull);
}

// Words of columns 4 * quad .. 4 * quad + 3 of mask row `row`.
__device__ __forceinline__ void philox(const DropParams& d, uint32_t quad, uint32_t row, uint64_t offset,
                                       uint32_t (&out)[4]) {
  uint32_t c0 = quad, c1 = row, c2 = static_cast<uint32_t>(offset), c3 = static_cast<uint32_t>(offset >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = static_cast<uint64_t>(kPhiloxM0) * c0;
    const uint64_t b = static_cast<uint64_t>(kPhiloxM1) * c2;
    c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ d.key[2 * r];
    c1 = static_cast<uint32_t>(b);
    c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ d.key[2 * r + 1];
    c3 = static_cast<uint32_t>(a);
  }
  out[0] = c0;
  out[1] = c1;
  out[2] = c2;
  out[3] = c3;
}

// Whether one element is kept (kernels that handle columns one by one).
__device__ __forceinline__ bool keep1(const DropParams& d, int64_t col, int64_t row, uint64_t offset) {
  uint32_t w[4];
  philox(d, static_cast<uint32_t>(col >> 2), static_cast<uint32_t>(d.row0 + row), offset, w);
  const uint32_t j = static_cast<uint32_t>(col) & 3u;
  return (j == 0 ? w[0] : j == 1 ? w[1] : j == 2 ? w[2] : w[3]) >= d.least;
}

// ---------------------------------------------------------------------------------------
// 8-bit values. The largest magnitude of a group is found with sm_100's three-input maximum
// of absolute values, in the form that keeps NaN; across lanes and warps it travels as its
// bits, which order as unsigned integers: below infinity, infinity below NaN.
// ---------------------------------------------------------------------------------------
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

__device__ __forceinline__ float largest8(float most, const float2 (&y)[4]) {
  most = max3_abs(most, y[0].x, y[0].y);
  most = max3_abs(most, y[1].x, y[1].y);
  most = max3_abs(most, y[2].x, y[2].y);
  return max3_abs(most, y[3].x, y[3].y);
}

__device__ __forceinline__ uint32_t magnitude(float y) { return __float_as_uint(y) & 0x7fffffffu; }

// scale = max(largest / Q, 2^-126), NaN kept: the floor keeps 1 / scale finite where the
// group is zero or below the normal numbers.
__device__ __forceinline__ float scale_of(float largest, float inv_q) {
  const float s = largest * inv_q;
  return s < 1.17549435e-38f ? 1.17549435e-38f : s;
}

// 1 / scale to the last place or the one before: a q that lies between two of its values
// within that error may take either.
__device__ __forceinline__ float inverse(float scale) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(scale));
  return r;
}

// The 8-bit types. largest * inverse(scale) is Q within two places, so an int8 never rounds to
// -128; e4m3 saturates. NaN becomes e4m3's NaN, or int8's 0 (its scale is NaN).
struct E4M3 {
  static constexpr float kInvQ = 1.f / 448.f;
  __device__ __forceinline__ static uint32_t pack4(float2 a, float2 b) {
    return __nv_cvt_float2_to_fp8x2(a, __NV_SATFINITE, __NV_E4M3) |
           static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(b, __NV_SATFINITE, __NV_E4M3)) << 16;
  }
};
struct I8 {
  static constexpr float kInvQ = 1.f / 127.f;
  __device__ __forceinline__ static uint32_t pack4(float2 a, float2 b) {
    const uint32_t lo = __byte_perm(__float2int_rn(a.x), __float2int_rn(a.y), 0x0040);
    const uint32_t hi = __byte_perm(__float2int_rn(b.x), __float2int_rn(b.y), 0x0040);
    return __byte_perm(lo, hi, 0x5410);
  }
};

__device__ __forceinline__ uint8_t q1(int dt, float v) {
  const float2 p = make_float2(v, 0.f);
  return static_cast<uint8_t>(dt == RMSNORM_B200_I8 ? I8::pack4(p, p) : E4M3::pack4(p, p));
}

__device__ __forceinline__ void store1_q(void* base, int dt, int64_t e, float v) {
  st1(static_cast<uint8_t*>(base) + e, q1(dt, v));
}

}  // namespace rmsb200
