// row_ring.cuh -- the skeleton of the fused row kernels: persistent row groups that stream
// their rows through shared-memory rings, row totals within a group and across a cluster.
//
//   * A CTA of up to 1024 threads holds `groups` row groups of G threads. A group owns a ring
//     of S units of its own and drifts freely: nothing but the total of a row ties its warps
//     together, and nothing ties the groups of a CTA.
//   * A unit is R whole rows, or KC of a row's K vector steps where a row would fill the
//     ring. It is filled by one TMA bulk copy per tensor. A warp that has taken a unit's
//     values into registers releases it; the last warp to do so issues the copy of the unit S
//     further on. So a row's second pass runs from registers while its slot loads again.
//   * A vector step is 8 consecutive columns a thread, G threads side by side.
//   * A row wider than a CTA holds is split over the C CTAs of a cluster; their totals go
//     through distributed shared memory.
//   * weight and bias are kept in shared memory in fp32, read once a kernel: the first and the
//     last four columns of a vector in an array each, so that neighbouring lanes read
//     neighbouring 16 bytes.
// Every wait is bounded (device_common.cuh).
#pragma once

#include "fused_common.cuh"

namespace rmsb200 {

constexpr int kRowWarps = 32;     // of a CTA, at most
constexpr int kMaxUnits = 128;    // ring units of a CTA
constexpr int kMaxRowCtas = 16;   // CTAs of a cluster
constexpr int kScaleAlign = 256;  // slices are multiples of it, so that no group of a scale is split

struct RowPlan {
  int32_t G, groups, S, R, KC, C;
  int32_t unit_shift;   // log2(units per row)
  int32_t slice;        // columns of a CTA's slice (the last CTA's may be shorter)
  uint32_t unit_bytes;
  uint32_t off[3];      // byte offset of tensor i in a unit
  int32_t bias;         // a bias follows the weight in shared memory
  int32_t scale_slots;  // words a group has twice after the barriers, for the scales of odd rows
  int64_t tiles;        // units of R rows
};

// Steps of a ring unit in the kernels with a built-in row group of g threads and four steps.
// Every unit costs each warp a wait and a release: at 1.3e8 elements, 16384 columns (g = 512)
// take 256 us in units of two steps (48 KB), 298 us of one; 8192 columns (g = 256) 237 us in
// units of four steps, 251 us of two.
__host__ __device__ constexpr int bwd_unit_steps(int g) { return g <= 256 ? 4 : 2; }

// Shared memory after the rings and the affine copies.
struct RowBars {
  uint64_t full[kMaxUnits];
  uint64_t xbar[2];
  uint64_t gbar[2][kRowWarps];  // [.][group]: a row's total within the group
  int done[kMaxUnits];
  float xpart[2][kMaxRowCtas][2];
  float red[2][kRowWarps][2];
  uint32_t tmem;  // address of the CTA's tensor memory (backward)
};

struct RowCtx {
  unsigned char* ring;  // this group's
  float* w;
  float* b;
  RowBars* bars;
  uint64_t* full;       // this group's
  int* done;
  int gid, gl, lane, warp, nwarps;  // group, thread in it, lane, warp of the CTA, warps of the group
  uint32_t rank;                    // CTA of the cluster
  int64_t slice0;                   // first column of the slice
  int ncols;                        // columns of the slice
  int64_t first, step;              // tiles of this group: first, first + step, ...
  int64_t units;                    // ring units of this group
  uint32_t reds;                    // reductions done (double buffering)
};

__device__ __forceinline__ uint32_t ring_bytes(const RowPlan& pl) {
  return static_cast<uint32_t>(pl.groups * pl.S) * pl.unit_bytes;
}

__device__ __forceinline__ RowCtx row_begin(const RowPlan& pl, int64_t N) {
  RowCtx c;
  unsigned char* smem = rmsb_dyn_smem;
  c.gid = threadIdx.x / pl.G;
  c.gl = threadIdx.x - c.gid * pl.G;
  c.lane = threadIdx.x & 31;
  c.warp = threadIdx.x >> 5;
  c.nwarps = pl.G >> 5;
  c.ring = smem + static_cast<size_t>(c.gid * pl.S) * pl.unit_bytes;
  c.w = reinterpret_cast<float*>(smem + ring_bytes(pl));
  c.b = c.w + pl.slice;
  c.bars = reinterpret_cast<RowBars*>(c.b + (pl.bias ? pl.slice : 0));
  c.full = c.bars->full + c.gid * pl.S;
  c.done = c.bars->done + c.gid * pl.S;
  c.rank = pl.C > 1 ? cluster_ctarank() : 0;
  c.slice0 = static_cast<int64_t>(c.rank) * pl.slice;
  c.ncols = static_cast<int>(min(static_cast<int64_t>(pl.slice), N - c.slice0));
  const int64_t clusters = gridDim.x / pl.C;
  c.first = blockIdx.x / pl.C + c.gid * clusters;
  c.step = clusters * pl.groups;
  c.units = c.first < pl.tiles ? (((pl.tiles - 1 - c.first) / c.step + 1) << pl.unit_shift) : 0;
  c.reds = 0;
  if (threadIdx.x == 0) {
    for (int i = 0; i < pl.groups * pl.S; ++i) {
      mbar_init(&c.bars->full[i], 1);
      c.bars->done[i] = 0;
    }
    mbar_init(&c.bars->xbar[0], 1);
    mbar_init(&c.bars->xbar[1], 1);
    for (int g = 0; g < pl.groups; ++g) {
      mbar_init(&c.bars->gbar[0][g], c.nwarps);
      mbar_init(&c.bars->gbar[1][g], c.nwarps);
    }
    fence_mbar_init();
  }
  __syncthreads();
  if (pl.C > 1) cluster_sync_all();  // every CTA's barriers stand before a peer signals them
  return c;
}

// weight (ones where absent) and bias of the slice, in fp32. Ends with a CTA barrier.
__device__ __forceinline__ void load_affine(const RowPlan& pl, const RowCtx& c, const void* w, int w_dt, const void* b,
                                            int b_dt) {
  const bool vec = (reinterpret_cast<uintptr_t>(w) & 15) == 0 && (reinterpret_cast<uintptr_t>(b) & 15) == 0;
  for (int v = threadIdx.x; v * 8 < c.ncols; v += blockDim.x) {
    float f[2][8];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const void* a = k == 0 ? w : b;
      const int dt = k == 0 ? w_dt : b_dt;
#pragma unroll
      for (int i = 0; i < 8; ++i) f[k][i] = 1.f;
      if (!a) continue;
      if (vec) {
        load8_rt(a, dt, c.slice0 + v * 8, f[k], true);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[k][i] = load1_rt(a, dt, c.slice0 + v * 8 + i);
      }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (k == 1 && !pl.bias) continue;
      float4* dst = reinterpret_cast<float4*>(k == 0 ? c.w : c.b) + v;
      dst[0] = make_float4(f[k][0], f[k][1], f[k][2], f[k][3]);
      dst[pl.slice / 8] = make_float4(f[k][4], f[k][5], f[k][6], f[k][7]);
    }
  }
  __syncthreads();
}

// Columns col .. col + 7 of an affine array (col a multiple of 8).
__device__ __forceinline__ void affine8(const RowPlan& pl, const float* a, int col, float2 (&v)[4]) {
  const float4 lo = reinterpret_cast<const float4*>(a)[col >> 3];
  const float4 hi = reinterpret_cast<const float4*>(a + pl.slice / 2)[col >> 3];
  v[0] = make_float2(lo.x, lo.y); v[1] = make_float2(lo.z, lo.w);
  v[2] = make_float2(hi.x, hi.y); v[3] = make_float2(hi.z, hi.w);
}

// Copies unit u of this group into its slot: kStreams tensors with elements of bytes[i].
template <int kStreams>
__device__ __forceinline__ void issue_unit(const RowPlan& pl, const RowCtx& c, int64_t u, int slot, int64_t rows,
                                           int64_t N, const void* (&src)[kStreams], const int (&bytes)[kStreams],
                                           uint64_t policy) {
  const int64_t row0 = (c.first + (u >> pl.unit_shift) * c.step) * pl.R;
  const int chunk = static_cast<int>(u) & ((1 << pl.unit_shift) - 1);
  const int width = pl.KC * pl.G * 8;
  const int col0 = chunk * width;
  int64_t elems;
  if (pl.R > 1)
    elems = min(static_cast<int64_t>(pl.R), rows - row0) * N;
  else
    elems = max(0, min(width, c.ncols - col0));
  uint64_t* bar = &c.full[slot];
  uint32_t total = 0;
#pragma unroll
  for (int i = 0; i < kStreams; ++i) total += static_cast<uint32_t>(elems) * bytes[i];
  if (total == 0) {
    mbar_arrive(bar);
    return;
  }
  mbar_arrive_expect_tx(bar, total);
  const int64_t e = row0 * N + c.slice0 + col0;
#pragma unroll
  for (int i = 0; i < kStreams; ++i)
    if (bytes[i])
      bulk_load(c.ring + static_cast<size_t>(slot) * pl.unit_bytes + pl.off[i],
                static_cast<const unsigned char*>(src[i]) + e * bytes[i], static_cast<uint32_t>(elems) * bytes[i], bar,
                policy);
}

// Every lane of a warp, after its last read of the slot. True on lane 0 of the group's last
// warp: it refills the slot. (Refilling when the row's total is complete, which needs no count,
// starts the copies later: 7 % slower with four warps a row or fewer.)
__device__ __forceinline__ bool release_unit(const RowCtx& c, int slot) {
  __syncwarp();
  if (c.lane != 0) return false;
  __threadfence_block();
  if (atomicAdd(&c.done[slot], 1) != c.nwarps - 1) return false;
  c.done[slot] = 0;
  __threadfence_block();
  fence_proxy_async_smem();
  return true;
}

// A row's sum and largest magnitude (bits) over the group's threads and the cluster's CTAs.
// Every thread gets the same bits: the warps' values are added in one shuffle tree in warp
// order, the CTAs' in rank order. `meanwhile` runs between a warp's contribution and its wait
// for the others': work that does not need the total.
// A warp writes slot k again two totals later, after it has taken the total in between; every
// warp contributed to that one after it had taken slot k.
// Across the cluster (one group a CTA), `xbar[k]` completes when the C CTAs' 8-byte contributions have landed
// (they may land before it is armed). A peer writes slot k again two totals later, when it has
// this CTA's contribution to the one in between; warp 0 sends that after every warp of this
// CTA has contributed to it, with slot k read.
template <bool kSum, bool kMax, typename F>
__device__ __forceinline__ void row_total(const RowPlan& pl, RowCtx& c, float& sum, uint32_t& most, int site,
                                          F&& meanwhile) {
  if (kSum) sum = warp_sum(sum);
  if (kMax) most = __reduce_max_sync(0xffffffffu, most);
  const uint32_t k = c.reds & 1u, parity = (c.reds >> 1) & 1u;
  if (pl.G > 32) {
    float(*red)[2] = c.bars->red[k];
    uint64_t* bar = &c.bars->gbar[k][c.gid];
    if (c.lane == 0) {
      if (kSum) red[c.warp][0] = sum;
      if (kMax) red[c.warp][1] = __uint_as_float(most);
      mbar_arrive(bar);
    }
    meanwhile();
    mbar_wait_warp(bar, parity, site);
    __syncwarp();
    const int w = c.gid * c.nwarps + c.lane;
    if (kSum) sum = warp_sum(c.lane < c.nwarps ? red[w][0] : 0.f);
    if (kMax) most = __reduce_max_sync(0xffffffffu, c.lane < c.nwarps ? __float_as_uint(red[w][1]) : 0u);
  } else {
    meanwhile();
  }
  if (pl.C > 1) {
    float(*part)[2] = c.bars->xpart[k];
    uint64_t* bar = &c.bars->xbar[k];
    if (c.warp == 0) {
      if (c.lane == 0) mbar_arrive_expect_tx(bar, static_cast<uint32_t>(pl.C) * 8u);
      if (c.lane < pl.C) {
        const uint32_t to_bar = map_peer(smem_u32(bar), c.lane);
        st_async_peer(map_peer(smem_u32(&part[c.rank][0]), c.lane), sum, to_bar);
        st_async_peer(map_peer(smem_u32(&part[c.rank][1]), c.lane), __uint_as_float(most), to_bar);
      }
    }
    mbar_wait_warp<true>(bar, parity, site);
    __syncwarp();
    if (kSum) sum = warp_sum(c.lane < pl.C ? part[c.lane][0] : 0.f);
    if (kMax) most = __reduce_max_sync(0xffffffffu, c.lane < pl.C ? __float_as_uint(part[c.lane][1]) : 0u);
  }
  ++c.reds;
}

template <bool kSum, bool kMax>
__device__ __forceinline__ void row_total(const RowPlan& pl, RowCtx& c, float& sum, uint32_t& most, int site) {
  row_total<kSum, kMax>(pl, c, sum, most, site, [] {});
}

// The end of a kernel: after a wait that ran out, the group's copies in flight land first; a
// CTA of a cluster stays until its peers no longer write to it.
__device__ __forceinline__ void row_end(const RowPlan& pl, const RowCtx& c) {
  if (c.gl == 0 && abort_requested())
    for (int s = 0; s < pl.S && s < c.units; ++s)
      mbar_wait(&c.full[s], static_cast<uint32_t>((c.units - 1 - s) / pl.S) & 1u, kSiteDrain, false);
  if (pl.C > 1) cluster_sync_all();
}

// The mask's words of columns col .. col + 7 (col a multiple of 8).
__device__ __forceinline__ void draw8(const DropParams& d, int64_t col, int64_t row, uint64_t offset,
                                      uint32_t (&w)[2][4]) {
  const uint32_t quad = static_cast<uint32_t>(col >> 2), mrow = static_cast<uint32_t>(d.row0 + row);
  philox(d, quad, mrow, offset, w[0]);
  philox(d, quad + 1, mrow, offset, w[1]);
}

// Kept values of `a`, `b` elsewhere.
__device__ __forceinline__ void select8(const DropParams& d, const uint32_t (&w)[2][4], const float2 (&a)[4],
                                        const float2 (&b)[4], float2 (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    v[2 * i].x = w[i][0] >= d.least ? a[2 * i].x : b[2 * i].x;
    v[2 * i].y = w[i][1] >= d.least ? a[2 * i].y : b[2 * i].y;
    v[2 * i + 1].x = w[i][2] >= d.least ? a[2 * i + 1].x : b[2 * i + 1].x;
    v[2 * i + 1].y = w[i][3] >= d.least ? a[2 * i + 1].y : b[2 * i + 1].y;
  }
}

}  // namespace rmsb200
