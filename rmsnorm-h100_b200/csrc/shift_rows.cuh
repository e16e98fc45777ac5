// shift_rows.cuh -- the fused row operators for contiguous rows of a width that no 16-byte
// vector divides, their tensors beginning on 16-byte boundaries.
//
// Element row * N of every tensor lies `lead` = row * N mod 8 elements past a boundary of eight
// elements, whatever the element's size. So a row is taken as the whole vectors that cover it,
// from `lead` elements before its first column on: copies, loads and stores are the aligned
// kernels' own, and only its first and last vector have elements of other rows to mask. The
// rows of one class modulo 8 (4, 2 where N divides by 2, 4) share their lead: a cluster works
// on one class, so that a thread keeps its columns from row to row and the affine parameters
// lie in shared memory at the row's offset. With 148 clusters a class has 18 or 19 of them,
// which costs 3 %. Measured at 1.3e8 elements (x, residual and outputs bf16, dropout), against
// the scalar accesses of odd_kernels.cuh: 4097 columns forward 354 / 592 us, backward 421 / 1372,
// 8 bits with a scale a row 240 / 531, a scale per 128 columns 396 / 531; 1001 columns 304 / 401,
// 389 / 787, 218 / 361, 344 / 361. Bound by instructions at 15 warps: for eight columns 389
// (dropout forward), 489 (backward), 458 (a scale per 128 columns), where the aligned kernels take
// 253, 304 and 200. The edges, a ninth more draws and the shuffles of their bits, and in the
// 8-bit forward a second total a row and the scales' way through shared memory make the rest.
#pragma once

#include <type_traits>

#include "row_ring.cuh"

namespace rmsb200 {

constexpr int kShiftThreads = 512;

// Rows of a cluster's class: c.first, c.first + c.step, ... as in RowCtx, with units of one row.
struct RowShift {
  int lead;
  int64_t end;  // N + lead: columns are counted from the vector that holds the row's first one
};

__device__ __forceinline__ RowShift shift_begin(const RowPlan& pl, RowCtx& c, int64_t rows, int64_t N) {
  const int period = 8 >> (__ffs(static_cast<int>(N & 7) | 8) - 1);
  const int64_t cluster = blockIdx.x / pl.C, clusters = gridDim.x / pl.C;
  const int64_t of_class = cluster & (period - 1);
  const int64_t mates = (clusters - of_class + period - 1) / period;
  RowShift sh;
  sh.lead = static_cast<int>((of_class * N) & 7);
  sh.end = N + sh.lead;
  c.first = of_class + period * (cluster / period + c.gid * mates);
  c.step = period * mates * pl.groups;
  c.units = c.first < rows ? (((rows - 1 - c.first) / c.step + 1) << pl.unit_shift) : 0;
  c.ncols = static_cast<int>(min(static_cast<int64_t>(pl.slice), sh.end - c.slice0));
  return sh;
}

// Weight (ones where absent) and bias at the row's offset, zeros beside the row. Ends with a CTA
// barrier.
__device__ __forceinline__ void shift_affine(const RowPlan& pl, const RowCtx& c, const RowShift& sh, const void* w,
                                             int w_dt, const void* b, int b_dt) {
  for (int i = threadIdx.x; i < pl.slice; i += blockDim.x) {
    const int64_t n = c.slice0 + i - sh.lead;
    const bool in = n >= 0 && c.slice0 + i < sh.end;
    const int at = (i & 4 ? pl.slice / 2 : 0) + (i >> 3) * 4 + (i & 3);  // as load_affine lays it out
    c.w[at] = in ? (w ? load1_rt(w, w_dt, n) : 1.f) : 0.f;
    if (pl.bias) c.b[at] = in ? load1_rt(b, b_dt, n) : 0.f;
  }
  __syncthreads();
}

// The tensor ends inside the unit's last vector: `size` shrinks to whole 16-byte granules within
// it, and the elements after them are moved one by one.
__device__ __noinline__ void shift_tail(const unsigned char* from, uint32_t have, int bytes, unsigned char* to,
                                        uint32_t* size) {
  *size = have & ~15u;
  for (uint32_t o = *size; o < have; o += bytes) {
    if (!RMSB_DBG_OK(from + o, bytes, kDbgScalarLoad)) continue;
    if (bytes == 4)
      *reinterpret_cast<uint32_t*>(to + o) = *reinterpret_cast<const uint32_t*>(from + o);
    else
      *reinterpret_cast<uint16_t*>(to + o) = *reinterpret_cast<const uint16_t*>(from + o);
  }
}

// As issue_unit, with the row's whole vectors. bytes[i] 0: tensor i is absent.
template <int kStreams>
__device__ __forceinline__ void shift_issue(const RowPlan& pl, const RowCtx& c, const RowShift& sh, int64_t u, int slot,
                                            int64_t rows, int64_t N, const void* (&src)[kStreams],
                                            const int (&bytes)[kStreams], uint64_t policy) {
  const int64_t row = c.first + (u >> pl.unit_shift) * c.step;
  const int width = pl.KC * pl.G * 8;
  const int col0 = (static_cast<int>(u) & ((1 << pl.unit_shift) - 1)) * width;
  const int elems = max(0, min(width, ((c.ncols + 7) & ~7) - col0));
  const int64_t e = row * N - sh.lead + c.slice0 + col0;
  unsigned char* slot_at = c.ring + static_cast<size_t>(slot) * pl.unit_bytes;
  uint64_t* bar = &c.full[slot];
  uint32_t size[kStreams], total = 0;
#pragma unroll
  for (int i = 0; i < kStreams; ++i) {
    size[i] = static_cast<uint32_t>(elems) * bytes[i];
    if (size[i] && e + elems > rows * N)
      shift_tail(static_cast<const unsigned char*>(src[i]) + e * bytes[i],
                 static_cast<uint32_t>(rows * N - e) * bytes[i], bytes[i], slot_at + pl.off[i], &size[i]);
    total += size[i];
  }
  if (total == 0) {
    mbar_arrive(bar);
    return;
  }
  mbar_arrive_expect_tx(bar, total);
#pragma unroll
  for (int i = 0; i < kStreams; ++i)
    if (size[i])
      bulk_load(slot_at + pl.off[i], static_cast<const unsigned char*>(src[i]) + e * bytes[i], size[i], bar, policy);
}

// A vector at column `col` (of RowShift's count): which of its elements belong to the row.
struct ShiftEdge {
  int lo, hi;  // elements lo .. hi - 1
  __device__ __forceinline__ ShiftEdge(const RowShift& sh, int64_t col)
      : lo(col == 0 ? sh.lead : 0), hi(static_cast<int>(min(static_cast<int64_t>(8), sh.end - col))) {}
  __device__ __forceinline__ bool whole() const { return lo == 0 && hi == 8; }
  __device__ __forceinline__ void mask(float2 (&v)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (2 * i < lo || 2 * i >= hi) v[i].x = 0.f;
      if (2 * i + 1 < lo || 2 * i + 1 >= hi) v[i].y = 0.f;
    }
  }
};

template <typename T>
__device__ __forceinline__ T shift_round(float v) {
  if constexpr (std::is_same_v<T, float>) return v;
  else if constexpr (std::is_same_v<T, __half>) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}

// Stores a vector at element e, those of its elements that belong to the row.
template <typename T>
__device__ __forceinline__ void shift_store(void* base, int64_t e, const ShiftEdge& edge, const float2 (&v)[4]) {
  T* p = static_cast<T*>(base) + e;
  if (edge.whole()) {
    Pair8<T>::store(p, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i >= edge.lo && i < edge.hi) st1(p + i, shift_round<T>(i & 1 ? v[i >> 1].y : v[i >> 1].x));
}

// T, or fp32 where that is asked for.
template <typename T>
__device__ __forceinline__ void shift_load(const unsigned char* p, bool f32, float2 (&v)[4]) {
  if (f32)
    Pair8<float>::load(p, v);
  else
    Pair8<T>::load(p, v);
}

// Keep decisions of a row: bit 8 j + i for element i of the lane's vector of step j < kSteps. A
// vector that begins within one of the generator's groups of four columns needs the first
// group of the next lane's too; those after a warp's last vectors are drawn together, the one
// of step j by lane j. All lanes of the warp call.
template <int kSteps>
__device__ __forceinline__ uint32_t shift_keep(const DropParams& d, const RowPlan& pl, const RowCtx& c,
                                               const RowShift& sh, int64_t row, uint64_t offset) {
  const uint32_t mrow = static_cast<uint32_t>(d.row0 + row);
  const int within = -sh.lead & 3;
  const int warp_col = (c.gl & ~31) * 8;
  const int64_t first = c.slice0 + warp_col - sh.lead;  // may be negative: bits of no meaning
  uint32_t w[4], after = 0, keep = 0;
  if (within) {
    philox(d, static_cast<uint32_t>((first + 256) >> 2) + c.lane * (pl.G * 2), mrow, offset, w);
#pragma unroll
    for (int i = 0; i < 4; ++i) after |= w[i] >= d.least ? 1u << i : 0u;
  }
#pragma unroll
  for (int j = 0; j < kSteps; ++j) {
    if (j * (pl.G * 8) + warp_col >= c.ncols) break;
    const uint32_t quad = static_cast<uint32_t>(first >> 2) + 2 * c.lane + j * (pl.G * 2);
    uint32_t bits = 0;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      philox(d, quad + k, mrow, offset, w);
#pragma unroll
      for (int i = 0; i < 4; ++i) bits |= w[i] >= d.least ? 1u << (4 * k + i) : 0u;
    }
    if (within) {
      const uint32_t next = __shfl_down_sync(0xffffffffu, bits, 1), last = __shfl_sync(0xffffffffu, after, j);
      bits = ((bits | (c.lane == 31 ? last : next) << 8) >> within) & 0xffu;
    }
    keep |= bits << (8 * j);
  }
  return keep;
}

}  // namespace rmsb200
