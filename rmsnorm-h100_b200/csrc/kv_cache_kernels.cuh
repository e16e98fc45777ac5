// kv_cache_kernels.cuh -- keys and values in 8 bits, in pages: written with a scale for every
// head of a token, and read back.
#pragma once

#include <type_traits>

#include "block_scale.cuh"

namespace rmsb200 {

constexpr int kSiteCacheSlot = 11;  // a slot beyond the cache
constexpr int kSiteCachePage = 12;  // a row whose page the cache or the table does not have

// Division of numbers below 2^31 by a divisor known on the host: n / d = n m >> (31 + l) with
// l = ceil(log2 d) and m = ceil(2^(31 + l) / d) (Granlund and Montgomery: Division by invariant
// integers using multiplication, 1994). The compiler's own take 20 instructions in 32 bits and
// over 100 in 64, of which every lane of a head makes two: half the time of a write.
struct Divisor {
  uint32_t m, shift, d;
};
inline Divisor divisor_of(uint32_t d) {
  uint32_t l = 0;
  while ((uint64_t{1} << l) < d) ++l;
  return {static_cast<uint32_t>(((uint64_t{1} << (31 + l)) + d - 1) / d), 31 + l, d};
}
__device__ __forceinline__ uint32_t divide(uint32_t n, const Divisor& d) {
  return static_cast<uint32_t>((static_cast<uint64_t>(n) * d.m) >> d.shift);
}

struct CacheSide {  // k or v
  unsigned char* data;
  int64_t page, slot, head;
  float* scales;
  int64_t s_page, s_slot, s_head;
  void* x;  // the tokens' heads: read by the write, written by the read
  int64_t x_token, x_head;
  bool vec_x, vec_q;
};

struct CacheParams {
  CacheSide side[2];
  int64_t pages, tokens;
  const void* slots;
  const int32_t* table;
  const int32_t* starts;
  int64_t table_width, table_stride;
  Divisor by_heads, by_page;
  int32_t sequences, page_size, heads, head_dim;
  bool slots_64bit, zero_rest;
  bool small;  // heads of all tokens, and slots of the cache, are fewer than 2^31
};

constexpr int kCacheThreads = 256;

template <typename X>
__device__ __forceinline__ float cache_load1(const void* base, int64_t e) {
  const X* p = static_cast<const X*>(base) + e;
  if (!RMSB_DBG_OK(p, sizeof(X), kDbgScalarLoad)) return 0.f;
  return static_cast<float>(*p);
}

// Item i is head i % heads of token i / heads.
__device__ __forceinline__ void cache_item(const CacheParams& p, int64_t i, int64_t* token, int32_t* head) {
  if (p.small) {
    const uint32_t t = divide(static_cast<uint32_t>(i), p.by_heads);
    *token = t;
    *head = static_cast<int32_t>(static_cast<uint32_t>(i) - t * p.by_heads.d);
  } else {
    *token = i / p.heads;
    *head = static_cast<int32_t>(i - *token * p.heads);
  }
}

// A head takes kLanes lanes of 8 values each; every one of them has kItems heads of k or of v
// (blockIdx.y) in flight.
//   scale = max(max |x| / Q, 2^-126), q = round(Q x / max |x|)
// Q x is exact for 16-bit x, and so is the quotient wherever it is a tie of q: 16-bit x lie on
// ties far more often than chance has it (one in 700 of normal bf16 values), which x / scale, or x
// times an inverse, would decide by the rounding of the scale. The quotient is the product with
// the inverse and one correction by its remainder (Markstein: Computation of elementary functions
// on the IBM RISC System/6000 processor, 1990), of numbers brought to max |x| in [1, 8) by a power
// of two, so that the remainder is exact. A head whose scale is 2^-126 takes x 2^126.
template <typename X, typename Q, int kLanes, int kItems>
__global__ void __launch_bounds__(kCacheThreads) cache_write_kernel(const __grid_constant__ CacheParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const CacheSide& side = blockIdx.y == 0 ? p.side[0] : p.side[1];
  constexpr int kGroups = kCacheThreads / kLanes;
  const int lane = threadIdx.x % kLanes, col = lane * 8;
  const int64_t items = p.tokens * p.heads;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (kGroups * kItems) + threadIdx.x / kLanes;
  float2 v[kItems][4];
  int64_t slot[kItems];
  int32_t head[kItems];
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    const int64_t i = first + j * kGroups;
    slot[j] = -1;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[j][k] = make_float2(0.f, 0.f);
    if (i >= items) continue;
    int64_t token;
    cache_item(p, i, &token, &head[j]);
    slot[j] = p.slots_64bit ? ld1(static_cast<const int64_t*>(p.slots) + token)
                            : ld1(static_cast<const int32_t*>(p.slots) + token);
    const int64_t e = token * side.x_token + head[j] * side.x_head + col;
    if (side.vec_x) {
      if (col < p.head_dim) Pair8<X>::load(static_cast<const X*>(side.x) + e, v[j]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (col + 2 * k < p.head_dim) v[j][k].x = cache_load1<X>(side.x, e + 2 * k);
        if (col + 2 * k + 1 < p.head_dim) v[j][k].y = cache_load1<X>(side.x, e + 2 * k + 1);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    uint32_t most = magnitude(largest8(0.f, v[j]));
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (slot[j] < 0) continue;
    if (slot[j] >= p.pages * p.page_size) {
      if (lane == 0) record_data_error(RMSNORM_B200_ERR_INVALID_ARGUMENT, kSiteCacheSlot);
      continue;
    }
    const int64_t page = p.small ? divide(static_cast<uint32_t>(slot[j]), p.by_page) : slot[j] / p.page_size;
    const int64_t place = slot[j] - page * p.page_size;
    constexpr float kTop = std::is_same<Q, I8>::value ? 127.f : 448.f;
    const float largest = __uint_as_float(most), s0 = __fdiv_rn(largest, kTop);
    const bool least = s0 < 1.17549435e-38f;  // NaN is not
    if (lane == 0)
      st1(side.scales + page * side.s_page + place * side.s_slot + head[j] * side.s_head, least ? 1.17549435e-38f : s0);
    if (col >= p.head_dim) continue;
    const int e = static_cast<int>(most >> 23);
    const float power = __uint_as_float(static_cast<uint32_t>(max(254 - e, 1)) << 23);
    const float times = least ? 8.5070592e37f : kTop * power;  // 2^126
    const float by = least ? 1.f : e < 255 ? largest * power : 0.f;  // infinity: no remainder
    const float inv = __frcp_rn(!least && e == 255 ? largest : by);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 n = mul2(v[j][k], splat2(times)), q = mul2(n, splat2(inv));
      v[j][k] = fma2(fma2(q, splat2(-by), n), splat2(inv), q);
    }
    const uint2 b = make_uint2(Q::pack4(v[j][0], v[j][1]), Q::pack4(v[j][2], v[j][3]));
    unsigned char* dst = side.data + page * side.page + place * side.slot + head[j] * side.head + col;
    if (side.vec_q) {
      if (RMSB_DBG_OK(dst, 8, kDbgVecStore)) *reinterpret_cast<uint2*>(dst) = b;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (col + k < p.head_dim) st1(dst + k, static_cast<unsigned char>((k < 4 ? b.x : b.y) >> (8 * (k & 3))));
    }
  }
}

template <typename Q>
__device__ __forceinline__ void unpack_octet(uint2 b, float s, float2 (&v)[4]);

template <>
__device__ __forceinline__ void unpack_octet<E4M3>(uint2 b, float s, float2 (&v)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const __nv_fp8x2_storage_t two = static_cast<__nv_fp8x2_storage_t>((k < 2 ? b.x : b.y) >> (16 * (k & 1)));
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(two, __NV_E4M3);
    v[k] = mul2(__half22float2(__half2(h)), splat2(s));
  }
}

template <>
__device__ __forceinline__ void unpack_octet<I8>(uint2 b, float s, float2 (&v)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t w = k < 2 ? b.x : b.y;
    v[k] = mul2(make_float2(static_cast<float>(static_cast<int8_t>(w >> (16 * (k & 1)))),
                            static_cast<float>(static_cast<int8_t>(w >> (16 * (k & 1) + 8)))),
                splat2(s));
  }
}

// Where a row of the packed sequences lies.
constexpr int32_t kRest = -1, kNowhere = -2;

__device__ __forceinline__ int2 cache_place(const CacheParams& p, int64_t token) {
  int32_t lo = 0, hi = p.sequences;  // the last start at or before the token is in [lo, hi]
  if (token >= ld1(p.starts + p.sequences)) return make_int2(kRest, 0);
  if (p.sequences == 0 || token < ld1(p.starts)) return make_int2(kNowhere, 0);
  while (hi - lo > 1) {
    const int32_t mid = lo + (hi - lo) / 2;
    if (token >= ld1(p.starts + mid)) lo = mid;
    else hi = mid;
  }
  // starts are 32 bits, and so are rows that lie before the last
  const uint32_t at = static_cast<uint32_t>(token - ld1(p.starts + lo)), column = at / static_cast<uint32_t>(p.page_size);
  if (static_cast<int64_t>(column) >= p.table_width) return make_int2(kNowhere, 0);
  const int32_t page = ld1(p.table + lo * p.table_stride + column);
  if (page < 0 || page >= p.pages) return make_int2(kNowhere, 0);
  return make_int2(page, static_cast<int32_t>(at - column * static_cast<uint32_t>(p.page_size)));
}

// A head takes kLanes lanes of 8 values; every one of them has kItems heads of k and as many of v
// in flight. The CTA's tokens are looked up first, a thread each.
template <typename X, typename Q, int kLanes, int kItems>
__global__ void __launch_bounds__(kCacheThreads) cache_read_kernel(const __grid_constant__ CacheParams p) {
  constexpr int kGroups = kCacheThreads / kLanes, kPer = kGroups * kItems;
  __shared__ int2 places[kPer];  // of the CTA's tokens: one at least for every head of the items
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x % kLanes, col = lane * 8;
  const int64_t items = p.tokens * p.heads, begin = static_cast<int64_t>(blockIdx.x) * kPer;
  int64_t token0, token1;
  int32_t unused;
  cache_item(p, begin, &token0, &unused);
  cache_item(p, min(begin + kPer, items) - 1, &token1, &unused);
  if (token0 + threadIdx.x <= token1) {
    const int2 at = cache_place(p, token0 + threadIdx.x);
    if (at.x == kNowhere) record_data_error(RMSNORM_B200_ERR_INVALID_ARGUMENT, kSiteCachePage);
    places[threadIdx.x] = at;
  }
  __syncthreads();
  uint2 b[kItems][2];
  float s[kItems][2];
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    const int64_t i = begin + j * kGroups + threadIdx.x / kLanes;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      b[j][k] = make_uint2(0, 0);
      s[j][k] = 0.f;
    }
    if (i >= items || col >= p.head_dim) continue;
    int64_t token;
    int32_t head;
    cache_item(p, i, &token, &head);
    const int2 at = places[token - token0];
    if (at.x < 0) {
      s[j][0] = s[j][1] = at.x == kNowhere ? __int_as_float(0x7fc00000) : 0.f;
      continue;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const CacheSide& side = p.side[k];
      const unsigned char* src = side.data + at.x * side.page + at.y * side.slot + head * side.head + col;
      s[j][k] = ld1(side.scales + at.x * side.s_page + at.y * side.s_slot + head * side.s_head);
      if (side.vec_q) {
        if (RMSB_DBG_OK(src, 8, kDbgVecLoad)) b[j][k] = *reinterpret_cast<const uint2*>(src);
      } else {
#pragma unroll
        for (int m = 0; m < 8; ++m)
          if (col + m < p.head_dim) {
            const uint32_t one = static_cast<uint32_t>(ld1(src + m)) << (8 * (m & 3));
            if (m < 4) b[j][k].x |= one;
            else b[j][k].y |= one;
          }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    const int64_t i = begin + j * kGroups + threadIdx.x / kLanes;
    if (i >= items || col >= p.head_dim) continue;
    int64_t token;
    int32_t head;
    cache_item(p, i, &token, &head);
    if (places[token - token0].x == kRest && !p.zero_rest) continue;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float2 v[4];
      unpack_octet<Q>(b[j][k], s[j][k], v);
      X* dst = static_cast<X*>(p.side[k].x) + i * p.head_dim + col;
      if (p.side[k].vec_x) {
        Pair8<X>::store(dst, v);
      } else {
#pragma unroll
        for (int m = 0; m < 8; ++m)
          if (col + m < p.head_dim) st1(dst + m, static_cast<X>(m & 1 ? v[m / 2].y : v[m / 2].x));
      }
    }
  }
}

}  // namespace rmsb200
