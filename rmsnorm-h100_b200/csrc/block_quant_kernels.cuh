// block_quant_kernels.cuh -- e4m3 values with a power of two as scale for 1 x 128 groups or
// 128 x 128 blocks, of x and of x transposed.
#pragma once

#include "block_scale.cuh"

namespace rmsb200 {

struct BlockQuantParams {
  const void* x;
  int64_t x_row;
  void* q;
  int64_t q_row;
  float* scales;
  int64_t scale_row, scale_group;
  void* q_t;
  int64_t q_t_row;
  float* scales_t;
  float* sum_part;  // [tile rows][cols]
  int64_t rows, cols;
  bool vec_in, vec_q, vec_t;  // 8-element vectors of x, 8-byte stores of q, 16-byte stores of q_t
  bool vec_all;               // all of those that there are
};

template <typename X>
__device__ __forceinline__ float load_one(const void* base, int64_t e) {
  const X* p = static_cast<const X*>(base) + e;
  if (!RMSB_DBG_OK(p, sizeof(X), kDbgScalarLoad)) return 0.f;
  if constexpr (sizeof(X) == 4) return *p;
  else return static_cast<float>(*p);
}

// Columns col .. col + 7 of a row at element e0; zeros from `cols` on.
template <typename X>
__device__ __forceinline__ void load_octet(const BlockQuantParams& p, int64_t e0, int64_t col, float2 (&v)[4]) {
  if (p.vec_in && col + 8 <= p.cols) {
    Pair8<X>::load(static_cast<const X*>(p.x) + e0 + col, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i].x = col + 2 * i < p.cols ? load_one<X>(p.x, e0 + col + 2 * i) : 0.f;
    v[i].y = col + 2 * i + 1 < p.cols ? load_one<X>(p.x, e0 + col + 2 * i + 1) : 0.f;
  }
}

__device__ __forceinline__ uint2 pack_octet(const float2 (&v)[4], float inv) {
  float2 t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) t[i] = mul2(v[i], splat2(inv));
  return make_uint2(E4M3::pack4(t[0], t[1]), E4M3::pack4(t[2], t[3]));
}

__device__ __forceinline__ void store_octet(const BlockQuantParams& p, int64_t row, int64_t col, uint2 b) {
  unsigned char* dst = static_cast<unsigned char*>(p.q) + row * p.q_row + col;
  if (p.vec_q && col + 8 <= p.cols) {
    if (RMSB_DBG_OK(dst, 8, kDbgVecStore)) *reinterpret_cast<uint2*>(dst) = b;
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (col + i < p.cols) st1(dst + i, static_cast<unsigned char>((i < 4 ? b.x : b.y) >> (8 * (i & 3))));
}

// Groups of a row, nothing else: 16 lanes a group, 8 columns a lane. One group a lane and many
// CTAs: four in flight a lane took 13.7 instead of 7.2 us for bf16, 2048 x 4096.
template <typename X>
__global__ void __launch_bounds__(256) quant_groups_kernel(const BlockQuantParams p, int64_t total, uint32_t groups) {
  pdl_launch_dependents();
  pdl_wait();
  const int at = (threadIdx.x & 15) * 8;
  const int64_t g = static_cast<int64_t>(blockIdx.x) * 16 + (threadIdx.x >> 4);
  const int64_t row = g / groups, group = g - row * groups;
  float2 v[4];
  if (g < total) {
    load_octet<X>(p, row * p.x_row, group * kBlock + at, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = make_float2(0.f, 0.f);
  }
  const uint32_t s = power_scale(largest_of<16>(octet_magnitude(v)));
  if (g >= total) return;
  if (at == 0) st1(p.scales + row * p.scale_row + group * p.scale_group, __uint_as_float(s));
  store_octet(p, row, group * kBlock + at, pack_octet(v, power_inverse(s)));
}

template <typename X>
__device__ __forceinline__ void load_held(const BlockQuantParams& p, int64_t row, int64_t col, Held<X>& h) {
  const X* src = static_cast<const X*>(p.x) + row * p.x_row + col;
  if (row < p.rows && p.vec_in && col + 8 <= p.cols) h.load(src);
  else h.load(src, row < p.rows ? p.cols - col : 0);
}

// One 128 x 128 tile a CTA, read once into registers: thread (warp w, lane l) holds rows
// 16 w + 8 (l / 16) + 0 .. 7 and columns 8 (l % 16) + 0 .. 7. Rows' groups lie in 16 lanes of one
// warp, columns' in all warps; the transposed bytes pass through shared memory, where the 8-byte
// piece of rows 8 u .. 8 u + 7 of column c lies at place u ^ (c / 8) of the column, so that
// neither side meets a bank twice.
// kWhole: a tile that lies inside the matrix, of tensors that allow vectors; without the checks of
// the others 4096 x 4096 in groups both ways take 16.3 instead of 22.0 us.
struct QuantShared {
  __align__(16) unsigned char turned[kBlock * kBlock];
  __align__(16) uint32_t col_most[8][kBlock];  // 16-bit values: two columns a word
  float col_sum[8][kBlock];
};

template <typename X, bool kBlocks, bool kWhole>
__device__ __forceinline__ void quant_tile(const BlockQuantParams& p, uint32_t tile_r, uint32_t tile_c, uint32_t tiles_c,
                                           QuantShared& sm) {
  auto& turned = sm.turned;
  auto& col_most = sm.col_most;
  auto& col_sum = sm.col_sum;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c8 = lane & 15, half = lane >> 4;
  const int64_t row0 = static_cast<int64_t>(tile_r) * kBlock + warp * 16 + half * 8;
  const int64_t col0 = static_cast<int64_t>(tile_c) * kBlock, col = col0 + c8 * 8;
  Held<X> h[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (kWhole) h[i].load(static_cast<const X*>(p.x) + row0 * p.x_row + col + i * p.x_row);
    else load_held<X>(p, row0 + i, col, h[i]);
  }
  if (p.sum_part) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float2 sum = h[0].pair(k);
#pragma unroll
      for (int i = 1; i < 8; ++i) sum = add2(sum, h[i].pair(k));
      sum.x += __shfl_xor_sync(0xffffffffu, sum.x, 16);
      sum.y += __shfl_xor_sync(0xffffffffu, sum.y, 16);
      if (half == 0) *reinterpret_cast<float2*>(&col_sum[warp][c8 * 8 + 2 * k]) = sum;
    }
  }
  float inv_t[8];  // of this thread's columns
  uint32_t most[8];
  if (kBlocks || p.q) most_of<X, 16, 8>(h, most);
  if (kBlocks) {
    uint32_t m = most[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) m = max(m, most[i]);
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 16));
    if (lane == 0) col_most[warp][0] = m;
    __syncthreads();
    uint32_t all = col_most[0][0];
#pragma unroll
    for (int w = 1; w < 8; ++w) all = max(all, col_most[w][0]);
    const uint32_t s = power_scale(all);
    const float inv = power_inverse(s);
    if (threadIdx.x == 0) {
      if (p.q) st1(p.scales + tile_r * p.scale_row + tile_c * p.scale_group, __uint_as_float(s));
      if (p.q_t) {
        st1(p.scales_t + static_cast<int64_t>(tile_r) * tiles_c + tile_c, __uint_as_float(s));
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) inv_t[k] = inv;
  }
  if (p.q) {
    unsigned char* dst = static_cast<unsigned char*>(p.q) + row0 * p.q_row + col;
    float* scale = p.scales + row0 * p.scale_row + tile_c * p.scale_group;
#pragma unroll
    for (int i = 0; i < 8; ++i, dst += p.q_row, scale += p.scale_row) {
      if (!kWhole && row0 + i >= p.rows) continue;
      float inv = inv_t[0];
      if (!kBlocks) {
        const uint32_t s = power_scale(most[i]);
        inv = power_inverse(s);
        if (c8 == 0) st1(scale, __uint_as_float(s));
      }
      const float2 v[4] = {h[i].pair(0), h[i].pair(1), h[i].pair(2), h[i].pair(3)};
      const uint2 b = pack_octet(v, inv);
      if constexpr (kWhole) {
        if (RMSB_DBG_OK(dst, 8, kDbgVecStore)) *reinterpret_cast<uint2*>(dst) = b;
      } else {
        store_octet(p, row0 + i, col, b);
      }
    }
  }
  if (!kBlocks && p.q_t) {
    if constexpr (sizeof(X) == 4) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i += 2)
          top = max3_abs(top, k & 1 ? h[i].v[k >> 1].y : h[i].v[k >> 1].x, k & 1 ? h[i + 1].v[k >> 1].y : h[i + 1].v[k >> 1].x);
        uint32_t m = magnitude(top);
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 16));
        if (half == 0) col_most[warp][c8 * 8 + k] = m;
      }
    } else {
      uint32_t m[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        m[k] = h[0].w[k] & 0x7fff7fffu;
#pragma unroll
        for (int i = 1; i < 8; ++i) m[k] = larger2(m[k], h[i].w[k] & 0x7fff7fffu);
        m[k] = larger2(m[k], __shfl_xor_sync(0xffffffffu, m[k], 16));
      }
      if (half == 0) *reinterpret_cast<uint4*>(&col_most[warp][c8 * 4]) = make_uint4(m[0], m[1], m[2], m[3]);
    }
    __syncthreads();
    uint32_t m[8];
    if constexpr (sizeof(X) == 4) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        m[k] = col_most[0][c8 * 8 + k];
#pragma unroll
        for (int w = 1; w < 8; ++w) m[k] = max(m[k], col_most[w][c8 * 8 + k]);
      }
    } else {
      uint4 t = *reinterpret_cast<const uint4*>(&col_most[0][c8 * 4]);
#pragma unroll
      for (int w = 1; w < 8; ++w) {
        const uint4 o = *reinterpret_cast<const uint4*>(&col_most[w][c8 * 4]);
        t = make_uint4(larger2(t.x, o.x), larger2(t.y, o.y), larger2(t.z, o.z), larger2(t.w, o.w));
      }
      const uint32_t two[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
      for (int k = 0; k < 8; ++k) m[k] = Held<X>::widen(k & 1 ? two[k / 2] >> 16 : two[k / 2] & 0xffffu);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t s = power_scale(m[k]);
      inv_t[k] = power_inverse(s);
      if (warp == 0 && half == 0 && (kWhole || col + k < p.cols)) st1(p.scales_t + tile_r * p.cols + col + k, __uint_as_float(s));
    }
  }
  if (p.q_t) {
    const int u = warp * 2 + half;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float2 t[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 a = h[2 * i].pair(k >> 1), b = h[2 * i + 1].pair(k >> 1);
        t[i] = k & 1 ? make_float2(a.y, b.y) : make_float2(a.x, b.x);
      }
      *reinterpret_cast<uint2*>(turned + (c8 * 8 + k) * kBlock + ((u ^ c8) << 3)) = pack_octet(t, inv_t[k]);
    }
  }
  __syncthreads();
  if (p.sum_part && threadIdx.x < kBlock && col0 + threadIdx.x < p.cols) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) sum += col_sum[w][threadIdx.x];
    st1(p.sum_part + static_cast<int64_t>(tile_r) * p.cols + col0 + threadIdx.x, sum);
  }
  if (!p.q_t) return;
  // eight lanes a column, 16 rows a lane
  const int64_t out0 = static_cast<int64_t>(tile_r) * kBlock + (threadIdx.x & 7) * 16;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = i * 32 + (threadIdx.x >> 3);
    if (!kWhole && (col0 + c >= p.cols || out0 >= p.rows)) continue;
    uint4 b = *reinterpret_cast<const uint4*>(turned + c * kBlock + (((threadIdx.x & 7) ^ (c >> 4)) << 4));
    if ((c >> 3) & 1) b = make_uint4(b.z, b.w, b.x, b.y);
    unsigned char* dst = static_cast<unsigned char*>(p.q_t) + (col0 + c) * p.q_t_row + out0;
    if (kWhole || (p.vec_t && out0 + 16 <= p.rows)) {
      if (RMSB_DBG_OK(dst, 16, kDbgVecStore)) *reinterpret_cast<uint4*>(dst) = b;
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const uint32_t word = j < 4 ? b.x : j < 8 ? b.y : j < 12 ? b.z : b.w;
        if (out0 + j < p.rows) st1(dst + j, static_cast<unsigned char>(word >> (8 * (j & 3))));
      }
    }
  }
}

template <typename X, bool kBlocks>
__global__ void __launch_bounds__(256, sizeof(X) == 4 ? 2 : 3) quant_tiles_kernel(const BlockQuantParams p, uint32_t tiles_c) {
  __shared__ QuantShared sm;
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t tile_r = blockIdx.x / tiles_c, tile_c = blockIdx.x - tile_r * tiles_c;
  if (p.vec_all && (tile_r + int64_t{1}) * kBlock <= p.rows && (tile_c + int64_t{1}) * kBlock <= p.cols)
    quant_tile<X, kBlocks, true>(p, tile_r, tile_c, tiles_c, sm);
  else
    quant_tile<X, kBlocks, false>(p, tile_r, tile_c, tiles_c, sm);
}

}  // namespace rmsb200
