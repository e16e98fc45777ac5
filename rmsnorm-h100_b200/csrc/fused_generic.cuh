// fused_generic.cuh -- parameters of the fused row operators, and their forward for rows wider
// than a cluster holds: one CTA per row, scalar accesses with types chosen at run time, the row
// read again from cache for each pass.
#pragma once

#include "fused_common.cuh"

namespace rmsb200 {

struct FusedFwdParams {
  const void* x;
  const void* res;
  const void* w;
  const void* b;
  void* out;        // floating output, or the 8-bit values
  void* ro;
  float* rstd;
  float* scales;    // null: floating output
  int64_t rows, N;
  int64_t scale_row, scale_group;
  int32_t x_dt, res_dt, w_dt, b_dt, out_dt, ro_dt;
  int32_t group;    // columns per scale (0 = the row)
  int32_t group_shift;  // its logarithm
  float eps;
  DropParams drop;
};

struct FusedBwdParams {
  const void* h;
  const void* dy;
  const float* rstd;
  const void* w;
  const void* dro;
  void* dx;
  void* dres;
  float* dw_part;
  float* db_part;
  int64_t rows, N;
  int32_t h_dt, dy_dt, w_dt, dro_dt, dx_dt, dres_dt;
  DropParams drop;
};

template <bool kDrop>
__device__ __forceinline__ float fused_h(const FusedFwdParams& p, int64_t row, int64_t n, uint64_t offset) {
  const int64_t e = row * p.N + n;
  float v = load1_rt(p.x, p.x_dt, e);
  if (kDrop) v = keep1(p.drop, n, row, offset) ? v * p.drop.scale : 0.f;
  if (p.res) v += load1_rt(p.res, p.res_dt, e);
  return v;
}

template <bool kDrop>
__global__ void __launch_bounds__(kGenericThreads) fused_fwd_generic_kernel(const FusedFwdParams p) {
  __shared__ float red[32];
  __shared__ uint32_t red_max[32];
  pdl_wait();
  const uint64_t offset = kDrop ? drop_offset(p.drop) : 0ull;
  const int64_t N = p.N;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool i8 = p.out_dt == RMSNORM_B200_I8;
  const float inv_q = i8 ? I8::kInvQ : E4M3::kInvQ;
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    float acc = 0.f;
    for (int64_t n = threadIdx.x; n < N; n += blockDim.x) {
      const float v = fused_h<kDrop>(p, r, n, offset);
      acc = fmaf(v, v, acc);
      if (p.ro) store1_rt(p.ro, p.ro_dt, r * N + n, v);
    }
    acc = block_sum_fixed(acc, red);
    const float rs = rsqrtf(acc / static_cast<float>(N) + p.eps);
    if (threadIdx.x == 0 && p.rstd) st1(&p.rstd[r], rs);
    auto y = [&](int64_t n) {
      const float w = p.w ? load1_rt(p.w, p.w_dt, n) : 1.f;
      const float b = p.b ? load1_rt(p.b, p.b_dt, n) : 0.f;
      return fmaf(fused_h<kDrop>(p, r, n, offset) * rs, w, b);
    };
    if (!p.scales) {
      for (int64_t n = threadIdx.x; n < N; n += blockDim.x) store1_rt(p.out, p.out_dt, r * N + n, y(n));
    } else if (p.group) {  // a warp per group
      for (int64_t g = warp; g * p.group < N; g += blockDim.x >> 5) {
        const int64_t end = min(N, (g + 1) * static_cast<int64_t>(p.group));
        uint32_t most = 0;
        for (int64_t n = g * p.group + lane; n < end; n += 32) most = max(most, magnitude(y(n)));
        const float s = scale_of(__uint_as_float(__reduce_max_sync(0xffffffffu, most)), inv_q);
        if (lane == 0) st1(&p.scales[r * p.scale_row + g * p.scale_group], s);
        for (int64_t n = g * p.group + lane; n < end; n += 32) store1_q(p.out, p.out_dt, r * N + n, y(n) * inverse(s));
      }
    } else {
      uint32_t most = 0;
      for (int64_t n = threadIdx.x; n < N; n += blockDim.x) most = max(most, magnitude(y(n)));
      most = __reduce_max_sync(0xffffffffu, most);
      if (lane == 0) red_max[warp] = most;
      __syncthreads();
      most = 0;
      for (int j = 0; j < static_cast<int>(blockDim.x >> 5); ++j) most = max(most, red_max[j]);
      __syncthreads();
      const float s = scale_of(__uint_as_float(most), inv_q);
      if (threadIdx.x == 0) st1(&p.scales[r * p.scale_row], s);
      for (int64_t n = threadIdx.x; n < N; n += blockDim.x) store1_q(p.out, p.out_dt, r * N + n, y(n) * inverse(s));
    }
  }
}

}  // namespace rmsb200
