// rope_kernels.cuh -- per-head RMSNorm of q and k with rotary positions, forward and backward.
#pragma once

#include <type_traits>

#include "device_common.cuh"

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

// Row of the table for the position at index `at`, or -1 where it lies outside the table.
__device__ __forceinline__ int64_t rope_row_at(const RopeParams& p, int64_t at) {
  const int64_t t = p.pos64 ? ld1(static_cast<const int64_t*>(p.pos) + at)
                            : static_cast<int64_t>(ld1(static_cast<const int32_t*>(p.pos) + at));
  if (t >= 0 && t < p.table_rows) return t;
  record_data_error(RMSNORM_B200_ERR_INVALID_ARGUMENT, kSiteRopePosition);
  return -1;
}

// The same for a pair of a token.
__device__ __forceinline__ int64_t rope_row(const RopeParams& p, int64_t token, int pair) {
  const int axis = static_cast<int>(p.axis_of[pair >> 5] >> (2 * (pair & 31))) & 3;
  return rope_row_at(p, axis * p.pos_axis + token);
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
// 16-byte granules.
//
// A lane owns two 4-element chunks of a head, chosen so that both columns of a pair are its
// own: a lane of the turned part has pairs 4l .. 4l + 3, that is columns 4l .. and
// 4l + rotary_dim / 2 .. (or 8l .. 8l + 7 when interleaved, pairs 4l .. 4l + 3 as well); a
// lane of the rest has eight neighbouring columns. So no value crosses lanes for the turn,
// and a lane needs only four cosines and four sines, which serve every head it works on.
// L = the smallest power of two with 8 L >= head_dim lanes hold a head; a warp holds 32 / L.
//
// A warp streams its heads of token after token through a ring in shared memory of its own
// (one bulk copy per tensor and token, or one per head where a token's heads are not
// neighbours), so it waits for nobody but its copies; what a token costs beyond its data
// (positions, table, addresses) is spread over the U heads of a lane and fetched ahead: the
// position two tokens, cosines and sines one.
// ---------------------------------------------------------------------------------------
template <typename T>
struct Chunk4 {
  uint2 v;
  static constexpr bool kB = std::is_same_v<T, __nv_bfloat16>;
  __device__ __forceinline__ void load(const void* p, int64_t e) {
    const T* q = static_cast<const T*>(p) + e;
    v = RMSB_DBG_OK(q, 8, kDbgVecLoad) ? *reinterpret_cast<const uint2*>(q) : make_uint2(0u, 0u);
  }
  __device__ __forceinline__ void get(float2* f) const {
    f[0] = kB ? unpack_bf16x2_pair(v.x) : unpack_f16x2_pair(v.x);
    f[1] = kB ? unpack_bf16x2_pair(v.y) : unpack_f16x2_pair(v.y);
  }
  __device__ __forceinline__ static void store(void* p, int64_t e, const float2* f) {
    T* q = static_cast<T*>(p) + e;
    const uint2 u = kB ? make_uint2(pack_bf16x2_pair(f[0]), pack_bf16x2_pair(f[1]))
                       : make_uint2(pack_f16x2_pair(f[0]), pack_f16x2_pair(f[1]));
    if (RMSB_DBG_OK(q, 8, kDbgVecStore)) __stcs(reinterpret_cast<uint2*>(q), u);
  }
};
template <>
struct Chunk4<float> {
  float4 v;
  __device__ __forceinline__ void load(const void* p, int64_t e) {
    const float* q = static_cast<const float*>(p) + e;
    v = RMSB_DBG_OK(q, 16, kDbgVecLoad) ? *reinterpret_cast<const float4*>(q) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __device__ __forceinline__ void get(float2* f) const {
    f[0] = make_float2(v.x, v.y);
    f[1] = make_float2(v.z, v.w);
  }
  __device__ __forceinline__ static void store(void* p, int64_t e, const float2* f) {
    float* q = static_cast<float*>(p) + e;
    if (RMSB_DBG_OK(q, 16, kDbgVecStore)) __stcs(reinterpret_cast<float4*>(q), make_float4(f[0].x, f[0].y, f[1].x, f[1].y));
  }
};

// A warp takes U * (32 / L) heads of a token, all of q or all of k, and keeps them over all
// the tokens it takes: the weight (and the backward's sums of its gradient) stay in registers.
// Where its heads are copied one by one, a lane each, it takes 32 at most.
struct RopePlan {
  int32_t S;            // ring slots of a warp
  uint32_t slot_bytes;  // of one tensor in a slot
  int32_t lanes_shift;  // log2(L)
  int32_t warp_heads;   // of a warp's share: a multiple of 32 / L
  int32_t jobs[2];      // warps' shares of a token: of q first, then of k
  int32_t turned_lanes; // lanes of the turned part: rotary_dim / 8
  int32_t cta_jobs;     // shares of a CTA, whose warps take warps / cta_jobs tokens at a time
};

struct RopeLane {
  int l, sub;     // lane within its head, head within the warp
  bool in;        // the lane has columns
  bool turned;
  int a, b;       // first columns of its chunks
};

template <bool kInterleaved>
__device__ __forceinline__ RopeLane rope_lane(const RopeParams& p, const RopePlan& pl) {
  RopeLane t;
  const int lane = threadIdx.x & 31;
  t.l = lane & ((1 << pl.lanes_shift) - 1);
  t.sub = lane >> pl.lanes_shift;
  t.in = t.l * 8 < p.D;
  t.turned = t.l < pl.turned_lanes;
  t.a = t.turned && !kInterleaved ? 4 * t.l : 8 * t.l;
  t.b = t.turned && !kInterleaved ? t.a + p.rd / 2 : t.a + 4;
  return t;
}

// The lane's four cosines and sines, a token ahead of their use, and the table row they come
// from a token before that. Where the four pairs have several axes, their rows are looked up
// with the cosines.
struct RopeTurn {
  float c[4], s[4];
  int32_t row;    // of the token after the one whose cosines are held; -1: outside the table
  int64_t first;  // the lane's axis in the positions
  bool one_axis;
  __device__ __forceinline__ RopeTurn(const RopeParams& p, const RopeLane& t, int64_t token, int64_t step) : row(-1) {
    const int i0 = 4 * t.l;
    const uint32_t axes = t.turned ? static_cast<uint32_t>(p.axis_of[i0 >> 5] >> (2 * (i0 & 31))) & 0xffu : 0u;
    one_axis = axes == (axes & 3u) * 0x55u;
    first = (axes & 3u) * p.pos_axis;
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = s[i] = 0.f;
    look_up(p, t, token);
    advance(p, t, token, token + step);
  }
  __device__ __forceinline__ void look_up(const RopeParams& p, const RopeLane& t, int64_t token) {
    if (t.turned && one_axis && token < p.tokens) row = static_cast<int32_t>(rope_row_at(p, first + token));
  }
  // Loads the cosines of `token` (whose row is held) and looks up the row of `after`.
  __device__ __forceinline__ void advance(const RopeParams& p, const RopeLane& t, int64_t token, int64_t after) {
    if (!t.turned || token >= p.tokens) return;
    const int i0 = 4 * t.l;
    if (!one_axis) {
#pragma unroll
      for (int i = 0; i < 4; ++i) rope_cos_sin(p, token, i0 + i, c[i], s[i]);
      return;
    }
    if (row >= 0) {
      const float* crow = p.table + static_cast<int64_t>(row) * p.rd + i0;
      const float* srow = crow + p.rd / 2;
      const float4 cv = RMSB_DBG_OK(crow, 16, kDbgVecLoad) ? __ldg(reinterpret_cast<const float4*>(crow)) : float4{};
      const float4 sv = RMSB_DBG_OK(srow, 16, kDbgVecLoad) ? __ldg(reinterpret_cast<const float4*>(srow)) : float4{};
      c[0] = cv.x; c[1] = cv.y; c[2] = cv.z; c[3] = cv.w;
      s[0] = sv.x; s[1] = sv.y; s[2] = sv.z; s[3] = sv.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = s[i] = __int_as_float(0x7fc00000);
    }
    look_up(p, t, after);
  }
};

// A token's cosines and sines as the turn uses them, the sines with both signs (the paired
// instructions negate no operand). sign -1 turns back.
struct RopeAngles {
  float2 c[2], s[2], n[2];
  __device__ __forceinline__ RopeAngles(const RopeTurn& t, bool back) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      c[i] = make_float2(t.c[2 * i], t.c[2 * i + 1]);
      const float2 plus = make_float2(t.s[2 * i], t.s[2 * i + 1]), minus = make_float2(-plus.x, -plus.y);
      s[i] = back ? minus : plus;
      n[i] = back ? plus : minus;
    }
  }
};

// y holds columns a .. a + 3, b .. b + 3, in pairs of neighbours.
template <bool kInterleaved>
__device__ __forceinline__ void rope_turn8(const RopeLane& t, const RopeAngles& r, float2 (&y)[4]) {
  if (!t.turned) return;
  if constexpr (kInterleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float c = i & 1 ? r.c[i >> 1].y : r.c[i >> 1].x, s = i & 1 ? r.s[i >> 1].y : r.s[i >> 1].x;
      y[i] = make_float2(y[i].x * c - y[i].y * s, y[i].y * c + y[i].x * s);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 u = y[i], v = y[2 + i];
      y[i] = fma2(v, r.n[i], mul2(u, r.c[i]));
      y[2 + i] = fma2(u, r.s[i], mul2(v, r.c[i]));
    }
  }
}

// Sums over the lanes of a head, of N values at once: their shuffles overlap.
template <int N>
__device__ __forceinline__ void rope_head_sums(float (&v)[N], int lanes_shift) {
  for (int o = 1 << lanes_shift >> 1; o > 0; o >>= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  }
}

__device__ __forceinline__ void rope_weight8(const RopeParams& p, int k, int64_t head, const RopeLane& t,
                                             float2 (&w)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = make_float2(1.f, 1.f);
  if (!p.w[k] || !t.in) return;
  const int64_t e = p.w_per_head[k] ? head * p.D : 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t at = e + (i < 2 ? t.a + 2 * i : t.b + 2 * i - 4);
    w[i] = make_float2(load1_rt(p.w[k], p.w_dt, at), load1_rt(p.w[k], p.w_dt, at + 1));
  }
}

// A warp's share of every token: its heads, and its first token and step.
struct RopeJob {
  bool works;
  int k, job, head0;     // q or k; share of it; the lane's first head
  int first;             // the warp's first head
  int per;               // heads of the warp side by side: the lane's next head is head0 + per
  int heads;
  int64_t token, step;
};

__device__ __forceinline__ RopeJob rope_job(const RopeParams& p, const RopePlan& pl, const RopeLane& t) {
  RopeJob b;
  const int warp = threadIdx.x >> 5;
  const int at_once = (blockDim.x >> 5) / pl.cta_jobs;  // tokens
  b.job = blockIdx.y * pl.cta_jobs + warp % pl.cta_jobs;
  b.works = b.job < pl.jobs[0] + pl.jobs[1];
  b.k = b.job >= pl.jobs[0];
  if (b.k) b.job -= pl.jobs[0];
  b.per = 32 >> pl.lanes_shift;
  b.first = b.job * pl.warp_heads;
  b.head0 = b.first + t.sub;
  b.heads = b.k ? p.heads[1] : p.heads[0];
  b.token = static_cast<int64_t>(blockIdx.x) * at_once + warp / pl.cta_jobs;
  b.step = static_cast<int64_t>(gridDim.x) * at_once;
  return b;
}

// Where the lane's heads lie in a tensor in global memory: its first head of the current token,
// moved on from token to token and from head to head.
template <typename T>
struct RopePlace {
  T* p;
  int64_t token_step, head_step;
  int da, db;
  __device__ __forceinline__ RopePlace(const RopeTensor& x, const RopeLane& t, const RopeJob& b)
      : p(static_cast<T*>(x.p) + b.token * x.ts + b.head0 * x.hs), token_step(b.step * x.ts), head_step(b.per * x.hs),
        da(t.a), db(t.b) {}
  __device__ __forceinline__ void load(const T* head, Chunk4<T> (&c)[2]) const {
    c[0].load(head, da);
    c[1].load(head, db);
  }
  __device__ __forceinline__ void store(T* head, const float2 (&y)[4]) const {
    Chunk4<T>::store(head, da, y);
    Chunk4<T>::store(head, db, y + 2);
  }
};

// A warp's ring: its heads of kTensors tensors (x, dy) for S tokens. Every lane of the warp
// calls. The forward keeps its source's address in registers (16384 tokens of 32 + 8 heads of 128,
// bf16: 69 against 77 us); the backward, short of them, makes addresses where a copy is issued
// (118 against 139 us).
template <typename T, int U, int kTensors>
struct RopeRing {
  uint32_t slots, full;  // byte offsets in shared memory of the warp's slots and barriers
  int slot;
  uint32_t phase;
  int64_t next;          // token to be copied next
  const T* src;          // forward: its first head of the warp
  __device__ __forceinline__ RopeRing(const RopeParams& p, const RopePlan& pl, const RopeJob& b) {
    const uint32_t warp = threadIdx.x >> 5, warps = blockDim.x >> 5, bytes = pl.S * kTensors * pl.slot_bytes;
    slots = warp * bytes;
    full = warps * bytes + warp * pl.S * 8;
    slot = 0;
    phase = 0;
    next = b.token;
    src = first_head(p, b, 0, next);
    if ((threadIdx.x & 31) == 0) {
      for (int s = 0; s < pl.S; ++s) mbar_init(bar(s), 1);
      fence_mbar_init();
    }
    __syncwarp();
  }
  __device__ __forceinline__ uint64_t* bar(int s) const { return reinterpret_cast<uint64_t*>(rmsb_dyn_smem + full) + s; }
  __device__ __forceinline__ const RopeTensor& tensor(const RopeParams& p, const RopeJob& b, int i) const {
    return i == 0 ? (b.k ? p.x[1] : p.x[0]) : (b.k ? p.dy[1] : p.dy[0]);
  }
  __device__ __forceinline__ const T* first_head(const RopeParams& p, const RopeJob& b, int i, int64_t token) const {
    const RopeTensor& x = tensor(p, b, i);
    return static_cast<const T*>(x.p) + token * x.ts + static_cast<int64_t>(b.first) * x.hs;
  }
  // Copies token `next` into slot s.
  __device__ __forceinline__ void issue(const RopeParams& p, const RopeJob& b, const RopePlan& pl, int s) {
    const int lane = threadIdx.x & 31;
    const int heads = min(pl.warp_heads, b.heads - b.first);
    if (next < p.tokens) {
      const uint64_t policy = l2_policy_evict_first();
      const uint32_t head_bytes = p.D * sizeof(T);
      if (lane == 0) mbar_arrive_expect_tx(bar(s), kTensors * heads * head_bytes);
      __syncwarp();
#pragma unroll
      for (int i = 0; i < kTensors; ++i) {
        const RopeTensor& x = tensor(p, b, i);
        unsigned char* dst = rmsb_dyn_smem + slots + (s * kTensors + i) * pl.slot_bytes;
        const T* from = kTensors == 1 ? src : first_head(p, b, i, next);
        const bool together = x.hs == p.D;
        if (lane < (together ? 1 : heads))  // heads apart: 32 at most
          bulk_load(dst + lane * head_bytes, from + lane * x.hs, together ? heads * head_bytes : head_bytes, bar(s),
                    policy);
        if (kTensors == 1) src += b.step * x.ts;
      }
    }
    next += b.step;
  }
  __device__ __forceinline__ void start(const RopeParams& p, const RopeJob& b, const RopePlan& pl) {
    for (int s = 0; s < pl.S; ++s) issue(p, b, pl, s);
  }
  __device__ __forceinline__ void wait(int site) {
    mbar_wait_warp(bar(slot), phase, site);
    __syncwarp();
  }
  // The lane's first head of the current token.
  __device__ __forceinline__ const T* held(const RopePlan& pl, const RopeParams& p, const RopeLane& t,
                                           int tensor) const {
    return reinterpret_cast<const T*>(rmsb_dyn_smem + slots + (slot * kTensors + tensor) * pl.slot_bytes) + t.sub * p.D;
  }
  // After the last load of a token: its slot takes the token S further on.
  __device__ __forceinline__ void advance(const RopeParams& p, const RopeJob& b, const RopePlan& pl) {
    __syncwarp();
    fence_proxy_async_smem();
    issue(p, b, pl, slot);
    if (++slot == pl.S) {
      slot = 0;
      phase ^= 1u;
    }
  }
  // After a wait that ran out: the copies in flight land before the warp leaves.
  __device__ __forceinline__ void drain(const RopeParams& p, const RopeJob& b, const RopePlan& pl) {
    __syncwarp();
    if (!abort_requested()) return;
    const int64_t n = b.token < p.tokens ? (p.tokens - 1 - b.token) / b.step + 1 : 0;
    for (int s = 0; s < pl.S && s < n; ++s)
      mbar_wait(bar(s), static_cast<uint32_t>((n - 1 - s) / pl.S) & 1u, kSiteDrain, false);
  }
};

struct RopeNoRing {
  __device__ __forceinline__ RopeNoRing(const RopeParams&, const RopePlan&, const RopeJob&) {}
};

template <typename T>
__device__ __forceinline__ void rope_get(const Chunk4<T> (&c)[2], float2 (&y)[4]) {
  c[0].get(y);
  c[1].get(y + 2);
}

// Warps of a CTA, at most. More of them have shallower rings and fewer registers: 16384 tokens of
// 32 + 8 heads of 128 take 72 us with 15 warps, 78 us with 20, 92 us with 25; backward 116, 120, 134.
constexpr int kRopeWarps = 16;

//   y = x rsqrt(mean(x^2) + eps) w;  a pair (y_a, y_b) becomes (y_a c - y_b s, y_b c + y_a s)
// kRing false: few tokens, whose heads a lane loads itself.
// 16384 tokens of 32 + 8 heads of 128, bf16, three axes: 71 us, 53 us of them bytes. Bound by
// instruction latency at 15 warps an SM: without positions and table it takes 60 us.
template <typename T, int U, bool kInterleaved, bool kNorm, bool kRing>
__global__ void __launch_bounds__(kRopeWarps * 32) rope_fwd_kernel(const RopeParams p, const RopePlan pl) {
  pdl_launch_dependents();
  pdl_wait();
  const RopeLane t = rope_lane<kInterleaved>(p, pl);
  const RopeJob b = rope_job(p, pl, t);
  if (!b.works) return;
  const int k = b.k;
  [[maybe_unused]] RopePlace<T> in(k ? p.x[1] : p.x[0], t, b);
  RopePlace<T> out(k ? p.out[1] : p.out[0], t, b);
  std::conditional_t<kRing, RopeRing<T, U, 1>, RopeNoRing> ring(p, pl, b);
  if constexpr (kRing) ring.start(p, b, pl);
  const bool per_head = p.w_per_head[k];
  const float inv_d = 1.f / static_cast<float>(p.D);
  const int mine = t.in ? (min(b.heads, b.first + pl.warp_heads) - b.head0 + b.per - 1) / b.per : 0;  // the lane has heads u < mine
  float2 w[4];
  RopeTurn turn(p, t, b.token, b.step);
  if (!per_head) rope_weight8(p, k, 0, t, w);
  for (int64_t token = b.token; token < p.tokens; token += b.step) {
    const T* head = in.p;
    int64_t head_step = in.head_step;
    if constexpr (kRing) {
      ring.wait(kSiteFwdFull);
      head = ring.held(pl, p, t, 0);
      head_step = b.per * p.D;
    }
    Chunk4<T> x[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u < mine)
        in.load(head + u * head_step, x[u]);
      else
        x[u][0].v = x[u][1].v = {};
    }
    if constexpr (kRing) ring.advance(p, b, pl);
    in.p += in.token_step;
    const RopeAngles angles(turn, false);
    turn.advance(p, t, token + b.step, token + 2 * b.step);
    float rs[U];
    if constexpr (kNorm) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float2 y[4];
        rope_get(x[u], y);
        float2 ss = mul2(y[0], y[0]);
#pragma unroll
        for (int i = 1; i < 4; ++i) ss = fma2(y[i], y[i], ss);
        rs[u] = ss.x + ss.y;
      }
      rope_head_sums(rs, pl.lanes_shift);
#pragma unroll
      for (int u = 0; u < U; ++u) rs[u] = rsqrtf(rs[u] * inv_d + p.eps);
    }
    T* to = out.p;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u < mine) {
        float2 y[4];
        rope_get(x[u], y);
        if constexpr (kNorm) {
#pragma unroll
          for (int i = 0; i < 4; ++i) y[i] = mul2(y[i], splat2(rs[u]));
        }
        if (per_head) rope_weight8(p, k, b.head0 + u * b.per, t, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = mul2(y[i], w[i]);
        rope_turn8<kInterleaved>(t, angles, y);
        out.store(to, y);
      }
      to += out.head_step;
    }
    out.p += out.token_step;
  }
  if constexpr (kRing) ring.drain(p, b, pl);
}

//   g = dout turned back;  dx = rstd (g w - xhat mean(xhat g w));  dweight = sum of g xhat
// 16384 tokens of 32 + 8 heads of 128, f16: 118 us, 78 us of them bytes: 243 instructions for
// eight columns, issued at half the SM's rate by 15 warps that the registers allow.
// The sums of dweight: a set per head the lane works on (kPerHead), or one set. The CTA adds
// its warps' sums in a fixed order and leaves one partial row: [q_heads + k_heads][head_dim]
// per blockIdx.x, or [q, k][head_dim] per CTA. A lane works on kBatch of its U heads at a time.
template <typename T, int U, int kBatch, bool kInterleaved, bool kNorm, bool kPerHead>
__global__ void __launch_bounds__(kRopeWarps * 32) rope_bwd_kernel(const RopeParams p, const RopePlan pl) {
  constexpr int kSets = kPerHead ? U : 1;
  static_assert(!kPerHead || U == kBatch, "sums of every head have registers of their own");
  __shared__ float sums[kRopeWarps][kRopeMaxDim];
  pdl_launch_dependents();
  pdl_wait();
  const RopeLane t = rope_lane<kInterleaved>(p, pl);
  const RopeJob b = rope_job(p, pl, t);
  const int warp = threadIdx.x >> 5;
  const int at_once = (blockDim.x >> 5) / pl.cta_jobs;
  const int first_job = blockIdx.y * pl.cta_jobs;
  const int all = pl.jobs[0] + pl.jobs[1];
  const int k = b.k, per = b.per;
  RopePlace<T> out(k ? p.out[1] : p.out[0], t, b);
  RopeRing<T, U, 2> ring(p, pl, b);
  if (b.works) ring.start(p, b, pl);
  const bool per_head = kPerHead && p.w_per_head[k];
  const float inv_d = 1.f / static_cast<float>(p.D);
  const int end = min(b.heads, b.first + pl.warp_heads);           // of the warp's heads
  const int mine = t.in ? (end - b.head0 + per - 1) / per : 0;     // the lane has heads u < mine
  const int used = (end - b.first + per - 1) / per;                // u < used: some lane of the warp has the head
  float2 acc[kSets][4], w[4];
#pragma unroll
  for (int i = 0; i < kSets; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[i][e] = make_float2(0.f, 0.f);
  // ones beside the head: 0 w of such a lane is part of the head's sums
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = make_float2(1.f, 1.f);
  if (!per_head) rope_weight8(p, k, 0, t, w);
  RopeTurn turn(p, t, b.works ? b.token : p.tokens, b.step);
  for (int64_t token = b.token; b.works && token < p.tokens; token += b.step) {
    ring.wait(kSiteBwdFull);
    const T* head_x = ring.held(pl, p, t, 0);
    const T* head_dy = ring.held(pl, p, t, 1);
    const RopeAngles angles(turn, true);
    turn.advance(p, t, token + b.step, token + 2 * b.step);
    T* to = out.p;
#pragma unroll 1
    for (int u0 = 0; u0 < used; u0 += kBatch) {
      Chunk4<T> x[kBatch][2], dy[kBatch][2];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (u0 + i < mine) {
          out.load(head_x + i * per * p.D, x[i]);
          out.load(head_dy + i * per * p.D, dy[i]);
        } else {
          x[i][0].v = x[i][1].v = dy[i][0].v = dy[i][1].v = {};
        }
      }
      head_x += kBatch * per * p.D;
      head_dy += kBatch * per * p.D;
      if (u0 + kBatch >= used) ring.advance(p, b, pl);
      // g = dout turned back; the sums of x^2 and x g w of all heads of the batch together
      float2 g[kBatch][4];
      float totals[2 * kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        rope_get(dy[i], g[i]);
        rope_turn8<kInterleaved>(t, angles, g[i]);
        if (u0 + i >= mine) {  // NaN cosines must not reach the sums of a lane without a head
#pragma unroll
          for (int e = 0; e < 4; ++e) g[i][e] = make_float2(0.f, 0.f);
        }
        if constexpr (kNorm) {
          if (per_head && u0 + i < mine) rope_weight8(p, k, b.head0 + (u0 + i) * per, t, w);
          float2 y[4];
          rope_get(x[i], y);
          float2 ss = mul2(y[0], y[0]), sg = mul2(y[0], mul2(g[i][0], w[0]));
#pragma unroll
          for (int e = 1; e < 4; ++e) {
            ss = fma2(y[e], y[e], ss);
            sg = fma2(y[e], mul2(g[i][e], w[e]), sg);
          }
          totals[2 * i] = ss.x + ss.y;
          totals[2 * i + 1] = sg.x + sg.y;
        }
      }
      if constexpr (kNorm) rope_head_sums(totals, pl.lanes_shift);
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (u0 + i < mine) {  // also for the sums: with eps 0 the rstd of no head is infinite
          if (per_head) rope_weight8(p, k, b.head0 + (u0 + i) * per, t, w);
          float2 y[4];
          rope_get(x[i], y);
          float rs = 1.f, m = 0.f;
          if constexpr (kNorm) {
            rs = rsqrtf(totals[2 * i] * inv_d + p.eps);
            m = -totals[2 * i + 1] * rs * inv_d;  // -mean of xhat g w
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float2& sum = acc[kPerHead ? i : 0][e];
            const float2 gw = mul2(g[i][e], w[e]);
            if constexpr (kNorm) {
              const float2 xhat = mul2(y[e], splat2(rs));
              sum = fma2(g[i][e], xhat, sum);
              y[e] = mul2(fma2(xhat, splat2(m), gw), splat2(rs));
            } else {
              sum = fma2(g[i][e], y[e], sum);
              y[e] = gw;
            }
          }
          out.store(to, y);
        }
        to += out.head_step;
      }
    }
    out.p += out.token_step;
  }
  if (b.works) ring.drain(p, b, pl);
  if (!p.part) return;
  // a lane's column of its sums' element i
  auto column = [&](int i) { return i < 4 ? t.a + i : t.b + i - 4; };
  auto value = [](const float2(&v)[4], int i) { return i & 1 ? v[i >> 1].y : v[i >> 1].x; };
  if constexpr (kPerHead) {
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (p.heads[0] + p.heads[1]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      __syncthreads();
      // a warp's 32 / L heads side by side, head_dim columns each
      if (t.in) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sums[warp][t.sub * p.D + column(i)] = value(acc[u], i);
      }
      __syncthreads();
      if (b.works && warp < pl.cta_jobs) {
        for (int i = threadIdx.x & 31; i < per * p.D; i += 32) {
          const int head = b.first + u * per + i / p.D;
          if (head >= end) continue;
          float v = 0.f;
          for (int j = 0; j < at_once; ++j) v += sums[warp + j * pl.cta_jobs][i];
          st1(&p.part[(row + (k ? p.heads[0] : 0) + head) * p.D + i % p.D], v);
        }
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      for (int o = 16; o >= 1 << pl.lanes_shift; o >>= 1) {
        acc[0][e].x += __shfl_xor_sync(0xffffffffu, acc[0][e].x, o);
        acc[0][e].y += __shfl_xor_sync(0xffffffffu, acc[0][e].y, o);
      }
    }
    if (t.in && t.sub == 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) sums[warp][column(i)] = value(acc[0], i);
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
