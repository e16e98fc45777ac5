// rope_kernels.cuh -- per-head RMSNorm of q and k with rotary positions, forward and backward.
#pragma once

#include <type_traits>

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

// ---------------------------------------------------------------------------------------
// Vectorised kernels: head_dim and rotary_dim multiples of 8, strides and addresses of whole
// 4-element chunks.
//
// A lane owns two 4-element chunks of a head, chosen so that both columns of a pair are its
// own: a lane of the turned part has pairs 4l .. 4l + 3, that is columns 4l .. and
// 4l + rotary_dim / 2 .. (or 8l .. 8l + 7 when interleaved, pairs 4l .. 4l + 3 as well); a
// lane of the rest has eight neighbouring columns. So no value crosses lanes for the turn,
// and a lane needs only four cosines and four sines, which serve every head it works on.
// L = the smallest power of two with 8 L >= head_dim lanes hold a head; a warp holds 32 / L.
// ---------------------------------------------------------------------------------------
constexpr int kRopeThreads = 256;

template <typename T>
struct Chunk4 {
  uint2 v;
  static constexpr bool kB = std::is_same_v<T, __nv_bfloat16>;
  __device__ __forceinline__ void load(const void* p, int64_t e) {
    const T* q = static_cast<const T*>(p) + e;
    v = RMSB_DBG_OK(q, 8, kDbgVecLoad) ? __ldcs(reinterpret_cast<const uint2*>(q)) : make_uint2(0u, 0u);
  }
  __device__ __forceinline__ void get(float* f) const {
    if constexpr (kB) {
      unpack_bf16x2(v.x, f[0], f[1]);
      unpack_bf16x2(v.y, f[2], f[3]);
    } else {
      unpack_f16x2(v.x, f[0], f[1]);
      unpack_f16x2(v.y, f[2], f[3]);
    }
  }
  __device__ __forceinline__ static void store(void* p, int64_t e, const float* f) {
    T* q = static_cast<T*>(p) + e;
    const uint2 u = kB ? make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]))
                       : make_uint2(pack_f16x2(f[0], f[1]), pack_f16x2(f[2], f[3]));
    if (RMSB_DBG_OK(q, 8, kDbgVecStore)) __stcs(reinterpret_cast<uint2*>(q), u);
  }
};
template <>
struct Chunk4<float> {
  float4 v;
  __device__ __forceinline__ void load(const void* p, int64_t e) {
    const float* q = static_cast<const float*>(p) + e;
    v = RMSB_DBG_OK(q, 16, kDbgVecLoad) ? __ldcs(reinterpret_cast<const float4*>(q)) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __device__ __forceinline__ void get(float* f) const { f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w; }
  __device__ __forceinline__ static void store(void* p, int64_t e, const float* f) {
    float* q = static_cast<float*>(p) + e;
    if (RMSB_DBG_OK(q, 16, kDbgVecStore)) __stcs(reinterpret_cast<float4*>(q), make_float4(f[0], f[1], f[2], f[3]));
  }
};

// Work of the vectorised kernels: a warp takes U * (32 / L) heads of one token, all of q or
// all of k: jobs 0 .. jobs[0] - 1 of a token are of q, the others of k.
struct RopePlan {
  int32_t lanes_shift;  // log2(L)
  int32_t jobs[2];      // of q and of k, per token
  int32_t turned_lanes; // lanes of the turned part: rotary_dim / 8
  int32_t cta_jobs;     // backward: jobs of a CTA, whose warps take warps / cta_jobs tokens at a time
};

struct RopeLane {
  int l, sub;     // lane within its head, head within the warp
  bool in;        // the lane has columns
  bool turned;
  int a, b;       // first columns of its chunks
};

__device__ __forceinline__ RopeLane rope_lane(const RopeParams& p, const RopePlan& pl) {
  RopeLane t;
  const int lane = threadIdx.x & 31;
  t.l = lane & ((1 << pl.lanes_shift) - 1);
  t.sub = lane >> pl.lanes_shift;
  t.in = t.l * 8 < p.D;
  t.turned = t.l < pl.turned_lanes;
  t.a = t.turned && !p.interleaved ? 4 * t.l : 8 * t.l;
  t.b = t.turned && !p.interleaved ? t.a + p.rd / 2 : t.a + 4;
  return t;
}

// The lane's four cosines and sines for a token.
__device__ __forceinline__ void rope_lane_turn(const RopeParams& p, const RopeLane& t, int64_t token, float (&c)[4],
                                               float (&s)[4]) {
  if (!t.turned) return;
  const int i0 = 4 * t.l;
  const uint32_t axis = static_cast<uint32_t>(p.axis_of[i0 >> 5] >> (2 * (i0 & 31))) & 0xffu;  // of four pairs
  if (axis == (axis & 3u) * 0x55u) {  // one axis for all four
    const int64_t r = rope_row(p, token, i0);
    if (r >= 0) {
      const float* row = p.table + r * p.rd + i0;
      const float4 cv = RMSB_DBG_OK(row, 16, kDbgVecLoad) ? __ldg(reinterpret_cast<const float4*>(row)) : float4{};
      const float* srow = row + p.rd / 2;
      const float4 sv = RMSB_DBG_OK(srow, 16, kDbgVecLoad) ? __ldg(reinterpret_cast<const float4*>(srow)) : float4{};
      c[0] = cv.x; c[1] = cv.y; c[2] = cv.z; c[3] = cv.w;
      s[0] = sv.x; s[1] = sv.y; s[2] = sv.z; s[3] = sv.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = s[i] = __int_as_float(0x7fc00000);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) rope_cos_sin(p, token, i0 + i, c[i], s[i]);
}

// y holds columns a .. a + 3, b .. b + 3. sign -1 turns back.
__device__ __forceinline__ void rope_turn8(const RopeParams& p, const RopeLane& t, const float (&c)[4],
                                           const float (&s)[4], float sign, float (&y)[8]) {
  if (!t.turned) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float sn = sign * s[i];
    if (p.interleaved) {
      const float u = y[2 * i], v = y[2 * i + 1];
      y[2 * i] = u * c[i] - v * sn;
      y[2 * i + 1] = v * c[i] + u * sn;
    } else {
      const float u = y[i], v = y[4 + i];
      y[i] = u * c[i] - v * sn;
      y[4 + i] = v * c[i] + u * sn;
    }
  }
}

__device__ __forceinline__ float rope_head_sum(float v, int lanes_shift) {
  for (int o = 1 << lanes_shift >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ void rope_weight8(const RopeParams& p, int k, int64_t head, const RopeLane& t,
                                             float (&w)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = 1.f;
  if (!p.w[k] || !t.in) return;
  const int64_t e = p.w_per_head[k] ? head * p.D : 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = load1_rt(p.w[k], p.w_dt, e + t.a + i);
    w[4 + i] = load1_rt(p.w[k], p.w_dt, e + t.b + i);
  }
}

template <typename T, int U>
__global__ void __launch_bounds__(kRopeThreads) rope_fwd_kernel(const RopeParams p, const RopePlan pl) {
  pdl_launch_dependents();
  pdl_wait();
  const RopeLane t = rope_lane(p, pl);
  const int per = 32 >> pl.lanes_shift;  // heads of a warp at a time
  const int jobs = pl.jobs[0] + pl.jobs[1];
  const int64_t work = p.tokens * jobs;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kRopeThreads / 32);
  const float inv_d = 1.f / static_cast<float>(p.D);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * (kRopeThreads / 32) + (threadIdx.x >> 5); i < work; i += step) {
    const int64_t token = i / jobs;
    int job = static_cast<int>(i - token * jobs);
    const int k = job >= pl.jobs[0];
    if (k) job -= pl.jobs[0];
    const int head0 = job * U * per + t.sub;
    Chunk4<T> x[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int head = head0 + u * per;
      if (t.in && head < p.heads[k]) {
        const int64_t e = token * p.x[k].ts + head * p.x[k].hs;
        x[u][0].load(p.x[k].p, e + t.a);
        x[u][1].load(p.x[k].p, e + t.b);
      } else {
        x[u][0].v = x[u][1].v = {};
      }
    }
    float c[4], s[4], w[8];
    rope_lane_turn(p, t, token, c, s);
    if (!p.w_per_head[k]) rope_weight8(p, k, 0, t, w);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int head = head0 + u * per;
      float y[8];
      x[u][0].get(y);
      x[u][1].get(y + 4);
      if (p.norm) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(y[e], y[e], ss);
        const float rs = rsqrtf(rope_head_sum(ss, pl.lanes_shift) * inv_d + p.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] *= rs;
      }
      if (t.in && head < p.heads[k]) {
        if (p.w_per_head[k]) rope_weight8(p, k, head, t, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] *= w[e];
        rope_turn8(p, t, c, s, 1.f, y);
        const int64_t o = token * p.out[k].ts + head * p.out[k].hs;
        Chunk4<T>::store(p.out[k].p, o + t.a, y);
        Chunk4<T>::store(p.out[k].p, o + t.b, y + 4);
      }
    }
  }
}

constexpr int kRopeBwdWarps = 16;

// A warp keeps its heads over all the tokens it takes, so the sums of dweight stay in its
// registers: a set per head it works on (kPerHead), or one set. The CTA adds its warps' sums
// in a fixed order and leaves one partial row: [q_heads + k_heads][head_dim] per blockIdx.x,
// or [q, k][head_dim] per CTA.
template <typename T, int U, bool kPerHead>
__global__ void __launch_bounds__(kRopeBwdWarps * 32) rope_bwd_kernel(const RopeParams p, const RopePlan pl) {
  constexpr int kSets = kPerHead ? U : 1;
  __shared__ float sums[kRopeBwdWarps][kRopeMaxDim];
  pdl_launch_dependents();
  pdl_wait();
  const RopeLane t = rope_lane(p, pl);
  const int per = 32 >> pl.lanes_shift;
  const int warp = threadIdx.x >> 5;
  const int at_once = (blockDim.x >> 5) / pl.cta_jobs;  // tokens
  const int all = pl.jobs[0] + pl.jobs[1];
  const int first_job = blockIdx.y * pl.cta_jobs;
  int job = first_job + warp % pl.cta_jobs;
  const bool works = job < all;
  const int k = job >= pl.jobs[0];
  if (k) job -= pl.jobs[0];
  const int head0 = job * U * per + t.sub;
  const float inv_d = 1.f / static_cast<float>(p.D);
  float acc[kSets][8], w[8];
#pragma unroll
  for (int i = 0; i < kSets; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[i][e] = 0.f;
  if (!p.w_per_head[k]) rope_weight8(p, k, 0, t, w);
  const int64_t step = static_cast<int64_t>(gridDim.x) * at_once;
  for (int64_t token = static_cast<int64_t>(blockIdx.x) * at_once + warp / pl.cta_jobs; works && token < p.tokens;
       token += step) {
    Chunk4<T> x[U][2], dy[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int head = head0 + u * per;
      if (t.in && head < p.heads[k]) {
        const int64_t d = token * p.dy[k].ts + head * p.dy[k].hs;
        dy[u][0].load(p.dy[k].p, d + t.a);
        dy[u][1].load(p.dy[k].p, d + t.b);
        const int64_t e = token * p.x[k].ts + head * p.x[k].hs;
        x[u][0].load(p.x[k].p, e + t.a);
        x[u][1].load(p.x[k].p, e + t.b);
      } else {
        x[u][0].v = x[u][1].v = dy[u][0].v = dy[u][1].v = {};
      }
    }
    float c[4], s[4];
    rope_lane_turn(p, t, token, c, s);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int head = head0 + u * per;
      const bool in = t.in && head < p.heads[k];
      float y[8], g[8];
      x[u][0].get(y);
      x[u][1].get(y + 4);
      dy[u][0].get(g);
      dy[u][1].get(g + 4);
      rope_turn8(p, t, c, s, -1.f, g);
      if (!in) {  // NaN cosines must not reach the sums of a lane without a head
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = 0.f;
      }
      if (p.w_per_head[k] && in) rope_weight8(p, k, head, t, w);
      float rs = 1.f, m = 0.f;
      if (p.norm) {
        float ss = 0.f, sg = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          ss = fmaf(y[e], y[e], ss);
          sg = fmaf(y[e], g[e] * w[e], sg);
        }
        ss = rope_head_sum(ss, pl.lanes_shift);
        sg = rope_head_sum(sg, pl.lanes_shift);
        rs = rsqrtf(ss * inv_d + p.eps);
        m = sg * rs * inv_d;  // mean of xhat g w
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float xhat = y[e] * rs;
        float& sum = acc[kPerHead ? u : 0][e];
        sum = fmaf(g[e], xhat, sum);
        y[e] = p.norm ? (g[e] * w[e] - xhat * m) * rs : g[e] * w[e];
      }
      if (in) {
        const int64_t o = token * p.out[k].ts + head * p.out[k].hs;
        Chunk4<T>::store(p.out[k].p, o + t.a, y);
        Chunk4<T>::store(p.out[k].p, o + t.b, y + 4);
      }
    }
  }
  if (!p.part) return;
  if constexpr (kPerHead) {
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (p.heads[0] + p.heads[1]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      __syncthreads();
      // a warp's 32 / L heads side by side, head_dim columns each
      if (t.in) {
        float* q = sums[warp] + t.sub * p.D;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          q[t.a + e] = acc[u][e];
          q[t.b + e] = acc[u][4 + e];
        }
      }
      __syncthreads();
      if (works && warp < pl.cta_jobs) {
        for (int i = threadIdx.x & 31; i < per * p.D; i += 32) {
          const int head = job * U * per + u * per + i / p.D;
          if (head >= p.heads[k]) continue;
          float v = 0.f;
          for (int j = 0; j < at_once; ++j) v += sums[warp + j * pl.cta_jobs][i];
          st1(&p.part[(row + (k ? p.heads[0] : 0) + head) * p.D + i % p.D], v);
        }
      }
    }
  } else {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = acc[0][e];
      for (int o = 16; o >= 1 << pl.lanes_shift; o >>= 1) v[e] += __shfl_xor_sync(0xffffffffu, v[e], o);
    }
    if (t.in && t.sub == 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sums[warp][t.a + e] = v[e];
        sums[warp][t.b + e] = v[4 + e];
      }
    }
    __syncthreads();
    float* row = p.part + (static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * 2 * p.D;
    for (int i = threadIdx.x; i < 2 * p.D; i += blockDim.x) {
      const int of_k = i >= p.D;
      float total = 0.f;
      for (int j = 0; j < static_cast<int>(blockDim.x >> 5); ++j) {
        const int jb = first_job + j % pl.cta_jobs;
        if (jb < all && (jb >= pl.jobs[0]) == of_k) total += sums[j][i - of_k * p.D];
      }
      st1(&row[i], total);
    }
  }
}

}  // namespace rmsb200
