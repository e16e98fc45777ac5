// rope_kernels.cuh -- per-head RMSNorm of q and k with rotary positions, forward and backward.
#pragma once

#include "device_common.cuh"
#include "generic_kernels.cuh"

namespace rmsb200 {

constexpr int kSiteRopePosition = 10;  // a position outside the table
constexpr int kRopeMaxDim = RMSNORM_B200_ROPE_MAX_HEAD_DIM;

struct RopeTensor {
  void* p;
  int64_t ts, hs;  // strides of a token and of a head, in elements
};

struct RopeParams {
  int64_t tokens, table_rows;
  const void* pos;
  int64_t pos_axis;
  const float* table;
  const void* w[2];        // of q and of k
  RopeTensor x[2];         // inputs
  RopeTensor dy[2];        // backward: gradients of the outputs
  RopeTensor out[2];       // outputs, or gradients of the inputs
  uint64_t axis_of[4];
  float* part;             // backward: partial rows of dweight, [chunks][q_heads + k_heads][head_dim], or null
  int32_t heads[2];
  int32_t w_per_head[2];
  int32_t D, rd, axes, interleaved, norm, pos64, dt, w_dt;
  float eps;
};

// Row of the table for pair i of a token, or -1 where the position lies outside it.
__device__ __forceinline__ int64_t rope_row(const RopeParams& p, int64_t token, int pair) {
  const int axis = static_cast<int>(p.axis_of[pair >> 5] >> (2 * (pair & 31))) & 3;
  const int64_t at = axis * p.pos_axis + token;
  const int64_t t = p.pos64 ? ld1(static_cast<const int64_t*>(p.pos) + at)
                            : static_cast<int64_t>(ld1(static_cast<const int32_t*>(p.pos) + at));
  if (t >= 0 && t < p.table_rows) return t;
  record_error(RMSNORM_B200_ERR_INVALID_ARGUMENT, kSiteRopePosition);
  return -1;
}

__device__ __forceinline__ void rope_cos_sin(const RopeParams& p, int64_t token, int pair, float& c, float& s) {
  const int64_t t = rope_row(p, token, pair);
  c = s = __int_as_float(0x7fc00000);
  if (t >= 0) {
    c = ld1(p.table + t * p.rd + pair);
    s = ld1(p.table + t * p.rd + p.rd / 2 + pair);
  }
}

// A warp per (token, head), scalar accesses: every head size, alignment and stride.
__global__ void __launch_bounds__(kGenericThreads) rope_fwd_generic_kernel(const RopeParams p) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int total = p.heads[0] + p.heads[1];
  const int64_t work = p.tokens * total;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5); i < work; i += step) {
    const int64_t token = i / total;
    int head = static_cast<int>(i % total);
    const int k = head >= p.heads[0];
    if (k) head -= p.heads[0];
    const int64_t e = token * p.x[k].ts + head * p.x[k].hs;
    const int64_t o = token * p.out[k].ts + head * p.out[k].hs;
    const int64_t we = p.w_per_head[k] ? static_cast<int64_t>(head) * p.D : 0;
    float rs = 1.f;
    if (p.norm) {
      float ss = 0.f;
      for (int d = lane; d < p.D; d += 32) {
        const float v = load1_rt(p.x[k].p, p.dt, e + d);
        ss = fmaf(v, v, ss);
      }
      rs = rsqrtf(warp_sum(ss) / static_cast<float>(p.D) + p.eps);
    }
    auto y = [&](int d) {
      const float v = load1_rt(p.x[k].p, p.dt, e + d) * rs;
      return p.w[k] ? v * load1_rt(p.w[k], p.w_dt, we + d) : v;
    };
    for (int j = lane; j < p.rd / 2; j += 32) {
      const int a = p.interleaved ? 2 * j : j, b = p.interleaved ? 2 * j + 1 : j + p.rd / 2;
      float c, s;
      rope_cos_sin(p, token, j, c, s);
      const float ya = y(a), yb = y(b);
      store1_rt(p.out[k].p, p.dt, o + a, ya * c - yb * s);
      store1_rt(p.out[k].p, p.dt, o + b, yb * c + ya * s);
    }
    for (int d = p.rd + lane; d < p.D; d += 32) store1_rt(p.out[k].p, p.dt, o + d, y(d));
  }
}

// One head per blockIdx.x, the tokens of chunk blockIdx.y a warp each; dweight is summed by
// the lane that owns the column, then over the warps in order.
__global__ void __launch_bounds__(kGenericThreads) rope_bwd_generic_kernel(const RopeParams p, int64_t chunk) {
  constexpr int kWarps = kGenericThreads / 32;
  __shared__ float acc[kWarps][kRopeMaxDim];
  __shared__ float g[kWarps][kRopeMaxDim];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int head = blockIdx.x;
  const int k = head >= p.heads[0];
  if (k) head -= p.heads[0];
  const int64_t we = p.w_per_head[k] ? static_cast<int64_t>(head) * p.D : 0;
  for (int d = lane; d < p.D; d += 32) acc[warp][d] = 0.f;
  __syncwarp();
  const int64_t end = min(p.tokens, (static_cast<int64_t>(blockIdx.y) + 1) * chunk);
  for (int64_t token = static_cast<int64_t>(blockIdx.y) * chunk + warp; token < end; token += kWarps) {
    const int64_t e = token * p.x[k].ts + head * p.x[k].hs;
    const int64_t de = token * p.dy[k].ts + head * p.dy[k].hs;
    const int64_t o = token * p.out[k].ts + head * p.out[k].hs;
    for (int j = lane; j < p.rd / 2; j += 32) {
      const int a = p.interleaved ? 2 * j : j, b = p.interleaved ? 2 * j + 1 : j + p.rd / 2;
      float c, s;
      rope_cos_sin(p, token, j, c, s);
      const float da = load1_rt(p.dy[k].p, p.dt, de + a), db = load1_rt(p.dy[k].p, p.dt, de + b);
      g[warp][a] = da * c + db * s;
      g[warp][b] = db * c - da * s;
    }
    for (int d = p.rd + lane; d < p.D; d += 32) g[warp][d] = load1_rt(p.dy[k].p, p.dt, de + d);
    __syncwarp();
    float ss = 0.f, sg = 0.f;
    auto w = [&](int d) { return p.w[k] ? load1_rt(p.w[k], p.w_dt, we + d) : 1.f; };
    if (p.norm) {
      for (int d = lane; d < p.D; d += 32) {
        const float v = load1_rt(p.x[k].p, p.dt, e + d);
        ss = fmaf(v, v, ss);
        sg = fmaf(v, g[warp][d] * w(d), sg);
      }
      ss = warp_sum(ss);
      sg = warp_sum(sg);
    }
    const float rs = p.norm ? rsqrtf(ss / static_cast<float>(p.D) + p.eps) : 1.f;
    const float c = p.norm ? sg * rs / static_cast<float>(p.D) : 0.f;
    for (int d = lane; d < p.D; d += 32) {
      const float xhat = load1_rt(p.x[k].p, p.dt, e + d) * rs;
      const float gd = g[warp][d];
      acc[warp][d] = fmaf(gd, xhat, acc[warp][d]);
      store1_rt(p.out[k].p, p.dt, o + d, p.norm ? (gd * w(d) - xhat * c) * rs : gd * w(d));
    }
    __syncwarp();
  }
  __syncthreads();
  if (!p.part) return;
  float* row = p.part + (static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * p.D;
  for (int d = threadIdx.x; d < p.D; d += blockDim.x) {
    float t = 0.f;
    for (int j = 0; j < kWarps; ++j) t += acc[j][d];
    st1(&row[d], t);
  }
}

}  // namespace rmsb200
