// kv_cache_kernels.cuh -- keys and values in 8 bits, in pages: written with a scale for every
// head of a token, and read back.
#pragma once

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
  Divisor by_rounds, by_page;  // rounds: of kItems heads, of a token
  int32_t sequences, page_size, heads, head_dim;
  bool slots_64bit, zero_rest;
  int32_t rounds;
  bool small;  // rounds of all tokens, and slots of the cache, are fewer than 2^31
};

constexpr int kCacheThreads = 256;

// Unit i is round i % rounds of token i / rounds.
__device__ __forceinline__ void cache_unit(const CacheParams& p, int64_t i, int64_t* token, int32_t* round) {
  if (p.small) {
    const uint32_t t = divide(static_cast<uint32_t>(i), p.by_rounds);
    *token = t;
    *round = static_cast<int32_t>(static_cast<uint32_t>(i) - t * p.by_rounds.d);
  } else {
    *token = i / p.rounds;
    *round = static_cast<int32_t>(i - *token * p.rounds);
  }
}

// A head takes kLanes lanes of kOctets times 8 values each; every one of them has kItems heads of a
// token's k or v (blockIdx.y) in flight, which share the work on its place (a head by itself takes
// 235 instructions for 8 values, 110 of them its place). Two octets a lane share the work on a
// head's scale as well: bf16, 16384 tokens of 8 heads of 128 19.9 us, with eight heads of one octet
// 23.8. Four CTAs an SM leave 64 registers; five (48, some in local memory) took 20.3 us.
//   scale = max(max |x| / Q, 2^-126), q = round(Q x / max |x|)
// Q x is exact for 16-bit x, and so is the quotient wherever it is a tie of q: 16-bit x lie on
// ties far more often than chance has it (one in 700 of normal bf16 values), which x / scale, or x
// times an inverse, would decide by the rounding of the scale. The quotient is the product with
// the inverse and one correction by its remainder (Markstein: Computation of elementary functions
// on the IBM RISC System/6000 processor, 1990), of numbers brought to max |x| in [1, 8) by a power
// of two, so that the remainder is exact. A head whose scale is 2^-126 takes x 2^126.
template <typename X, typename Q, int kLanes, int kItems, int kOctets>
__global__ void __launch_bounds__(kCacheThreads, kOctets == 2 ? 4 : 1) cache_write_kernel(const __grid_constant__ CacheParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const CacheSide& side = blockIdx.y == 0 ? p.side[0] : p.side[1];
  constexpr int kGroups = kCacheThreads / kLanes;
  const int lane = threadIdx.x % kLanes, col = lane * 8;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kGroups + threadIdx.x / kLanes;
  Held<X> held[kItems * kOctets];
  int64_t slot = -1, token = 0;
  int32_t round = 0;
  if (unit < p.tokens * p.rounds) {
    cache_unit(p, unit, &token, &round);
    slot = p.slots_64bit ? ld1(static_cast<const int64_t*>(p.slots) + token)
                         : ld1(static_cast<const int32_t*>(p.slots) + token);
  }
  const int32_t head0 = round * kItems, heads = unit < p.tokens * p.rounds ? min(kItems, p.heads - head0) : 0;
  const X* src = static_cast<const X*>(side.x) + token * side.x_token + head0 * side.x_head + col;
#pragma unroll
  for (int j = 0; j < kItems; ++j, src += side.x_head) {
#pragma unroll
    for (int o = 0; o < kOctets; ++o) {
      Held<X>& h = held[j * kOctets + o];
      const int at = o * kLanes * 8;
      h.zero();
      if (j >= heads || col + at >= p.head_dim) continue;
      if (side.vec_x) h.load(src + at);
      else h.load(src + at, p.head_dim - col - at);
    }
  }
  // no lane leaves before the last shuffle: its slot may differ from its neighbours'
  const bool beyond = slot >= p.pages * p.page_size;
  if (beyond && lane == 0 && head0 == 0) record_data_error(RMSNORM_B200_ERR_INVALID_ARGUMENT, kSiteCacheSlot);
  const bool kept = slot >= 0 && !beyond;
  const int64_t page = !kept ? 0 : p.small ? divide(static_cast<uint32_t>(slot), p.by_page) : slot / p.page_size;
  const int64_t place = kept ? slot - page * p.page_size : 0;
  float* scale = side.scales + page * side.s_page + place * side.s_slot + head0 * side.s_head;
  unsigned char* dst = side.data + page * side.page + place * side.slot + head0 * side.head + col;
  uint32_t largest_bits[kItems];
  most_of<X, kLanes, kItems, kOctets>(held, largest_bits);
  if (!kept) return;
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    if (j >= heads) break;
    constexpr float kTop = std::is_same<Q, I8>::value ? 127.f : 448.f, kInvTop = 1.f / kTop;
    const float largest = __uint_as_float(largest_bits[j]);
    const int e = static_cast<int>(largest_bits[j] >> 23);
    // max |x| / Q by the same correction, which infinity does not survive
    float s0 = largest * kInvTop;
    s0 = e == 255 ? largest : fmaf(fmaf(-s0, kTop, largest), kInvTop, s0);
    const bool least = s0 < 1.17549435e-38f;  // NaN is not
    if (lane == 0) st1(scale + j * side.s_head, least ? 1.17549435e-38f : s0);
    const float power = __uint_as_float(static_cast<uint32_t>(max(254 - e, 1)) << 23);
    const float times = least ? 8.5070592e37f : kTop * power;  // 2^126
    const float by = least ? 1.f : e < 255 ? largest * power : 0.f;  // infinity: no remainder
    const float inv = inverse(!least && e == 255 ? largest : by);
#pragma unroll
    for (int o = 0; o < kOctets; ++o) {
      const int at = o * kLanes * 8;
      if (col + at >= p.head_dim) continue;
      float2 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 n = mul2(held[j * kOctets + o].pair(k), splat2(times)), q = mul2(n, splat2(inv));
        v[k] = fma2(fma2(q, splat2(-by), n), splat2(inv), q);
      }
      const uint2 b = make_uint2(Q::pack4(v[0], v[1]), Q::pack4(v[2], v[3]));
      unsigned char* to = dst + j * side.head + at;
      if (side.vec_q) {
        if (RMSB_DBG_OK(to, 8, kDbgVecStore)) *reinterpret_cast<uint2*>(to) = b;
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (col + at + k < p.head_dim) st1(to + k, static_cast<unsigned char>((k < 4 ? b.x : b.y) >> (8 * (k & 3))));
      }
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

// A head takes kLanes lanes of 8 values; every one of them has kItems heads of a token's k and as
// many of its v in flight. The CTA's tokens are looked up first, a thread each.
template <typename X, typename Q, int kLanes, int kItems>
__global__ void __launch_bounds__(kCacheThreads) cache_read_kernel(const __grid_constant__ CacheParams p) {
  constexpr int kGroups = kCacheThreads / kLanes;
  __shared__ int2 places[kGroups];  // of the CTA's tokens: no more than its units
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x % kLanes, col = lane * 8;
  const int64_t units = p.tokens * p.rounds, begin = static_cast<int64_t>(blockIdx.x) * kGroups;
  const int64_t unit = min(begin + threadIdx.x / kLanes, units - 1);
  int64_t token0, token1, token;
  int32_t round;
  cache_unit(p, begin, &token0, &round);
  cache_unit(p, min(begin + kGroups, units) - 1, &token1, &round);
  if (token0 + threadIdx.x <= token1) {
    const int2 at = cache_place(p, token0 + threadIdx.x);
    if (at.x == kNowhere) record_data_error(RMSNORM_B200_ERR_INVALID_ARGUMENT, kSiteCachePage);
    places[threadIdx.x] = at;
  }
  cache_unit(p, unit, &token, &round);
  __syncthreads();
  if (begin + threadIdx.x / kLanes >= units || col >= p.head_dim) return;
  const int2 at = places[token - token0];
  if (at.x == kRest && !p.zero_rest) return;
  const int32_t head0 = round * kItems, heads = min(kItems, p.heads - head0);
  uint2 b[2][kItems];
  float s[2][kItems];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const CacheSide& side = p.side[k];
    const int64_t page = max(at.x, 0), place = at.y;
    const unsigned char* src = side.data + page * side.page + place * side.slot + head0 * side.head + col;
    const float* scale = side.scales + page * side.s_page + place * side.s_slot + head0 * side.s_head;
#pragma unroll
    for (int j = 0; j < kItems; ++j, src += side.head) {
      b[k][j] = make_uint2(0, 0);
      s[k][j] = at.x == kNowhere ? __int_as_float(0x7fc00000) : 0.f;
      if (at.x < 0 || j >= heads) continue;
      s[k][j] = ld1(scale + j * side.s_head);
      if (side.vec_q) {
        if (RMSB_DBG_OK(src, 8, kDbgVecLoad)) b[k][j] = *reinterpret_cast<const uint2*>(src);
      } else {
#pragma unroll
        for (int m = 0; m < 8; ++m)
          if (col + m < p.head_dim) {
            const uint32_t one = static_cast<uint32_t>(ld1(src + m)) << (8 * (m & 3));
            if (m < 4) b[k][j].x |= one;
            else b[k][j].y |= one;
          }
      }
    }
  }
  const int64_t e = token * p.side[0].x_token + head0 * p.head_dim + col;  // both outputs are contiguous
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    X* dst = static_cast<X*>(p.side[k].x) + e;
#pragma unroll
    for (int j = 0; j < kItems; ++j, dst += p.head_dim) {
      if (j >= heads) continue;
      float2 v[4];
      unpack_octet<Q>(b[k][j], s[k][j], v);
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
