// odd_kernels.cuh -- the fused row operators where the aligned and the shifted vector kernels
// (shift_rows.cuh) do not apply: tensors that begin off a 16-byte boundary, combinations of types
// without a kernel of their own, scales of column groups in rows of an odd width that take a
// cluster.
//
// The rows stream through the same rings: a bulk copy brings the aligned 16-byte granules
// that cover a unit, and the threads read the unit from its offset in the first of them. A
// granule that would leave the tensor at its very beginning or end is not copied; the
// issuing thread moves those elements itself. A lane then owns every 32nd column of its
// warp's 256 (not 8 in a row), so that scalar accesses to shared and global memory are
// consecutive across the warp at any alignment; their number bounds the kernel (1.3e8 bf16
// elements: forward 592 us, backward 1372 us at 4097 columns). Types are fixed at compile time
// where x, the residual and the output share one and residual_out has it or fp32; other
// combinations (Any) choose at run time, once a vector.
#pragma once

#include <type_traits>

#include "fused_generic.cuh"
#include "row_ring.cuh"

namespace rmsb200 {

constexpr int kOddThreads = 512;
constexpr int kOddSteps = 4;     // vector steps a thread at most: forward
constexpr int kOddBwdSteps = 2;  // backward

// One tensor that streams through the ring.
struct OddStream {
  const void* p;
  int dt, bytes;
};

// Byte offset in the slot of the unit's first element (address `a`).
__device__ __forceinline__ uint32_t odd_lead(const void* a) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>(a) & 15u);
}

// First element and number of elements of unit u.
__device__ __forceinline__ int64_t odd_unit(const RowPlan& pl, const RowCtx& c, int64_t u, int64_t rows, int64_t N,
                                            int64_t* elems) {
  const int64_t row0 = (c.first + (u >> pl.unit_shift) * c.step) * pl.R;
  const int chunk = static_cast<int>(u) & ((1 << pl.unit_shift) - 1);
  const int width = pl.KC * pl.G * 8;
  const int col0 = chunk * width;
  *elems = pl.R > 1 ? min(static_cast<int64_t>(pl.R), rows - row0) * N : max(0, min(width, c.ncols - col0));
  return row0 * N + c.slice0 + col0;
}

// The granules of `bytes` of elements at `begin` that lie within the tensor [base, limit): those
// outside are shrunk away, and their elements moved one by one to `dst` (the slot's address of
// the first granule). Only a tensor's first and last rows come here.
__device__ __noinline__ void odd_edges(uintptr_t base, uintptr_t limit, uintptr_t begin, uintptr_t end, int size,
                                       unsigned char* dst, uintptr_t* lo, uintptr_t* hi) {
  if (*lo < base) *lo += 16;
  if (*hi > limit) *hi -= 16;
  for (uintptr_t a = begin; a < end; a += size) {
    if (a >= *lo && a < *hi) {
      a = *hi - size;
      continue;
    }
    const void* from = reinterpret_cast<const void*>(a);
    if (!RMSB_DBG_OK(from, size, kDbgScalarLoad)) continue;
    unsigned char* to = dst + (begin & 15) + (a - begin);
    if (size == 4)
      *reinterpret_cast<uint32_t*>(to) = *static_cast<const uint32_t*>(from);
    else
      *reinterpret_cast<uint16_t*>(to) = *static_cast<const uint16_t*>(from);
  }
}

template <int kStreams>
__device__ __forceinline__ void odd_issue(const RowPlan& pl, const RowCtx& c, int64_t u, int slot, int64_t rows,
                                          int64_t N, const OddStream (&src)[kStreams], uint64_t policy) {
  int64_t elems;
  const int64_t e = odd_unit(pl, c, u, rows, N, &elems);
  uint64_t* bar = &c.full[slot];
  unsigned char* slot_at = c.ring + static_cast<size_t>(slot) * pl.unit_bytes;
  uintptr_t lo[kStreams], hi[kStreams];
  uint32_t off[kStreams];  // in the slot, of the first copied granule
  uint32_t total = 0;
#pragma unroll
  for (int i = 0; i < kStreams; ++i) {
    lo[i] = hi[i] = 0;
    if (!src[i].p || elems == 0) continue;
    const uintptr_t base = reinterpret_cast<uintptr_t>(src[i].p);
    const uintptr_t begin = base + e * src[i].bytes, end = begin + elems * src[i].bytes;
    const uintptr_t first = begin & ~static_cast<uintptr_t>(15), limit = base + rows * N * src[i].bytes;
    lo[i] = first;
    hi[i] = (end + 15) & ~static_cast<uintptr_t>(15);
    if (lo[i] < base || hi[i] > limit)
      odd_edges(base, limit, begin, end, src[i].bytes, slot_at + pl.off[i], &lo[i], &hi[i]);
    off[i] = pl.off[i] + static_cast<uint32_t>(lo[i] - first);
    if (hi[i] > lo[i]) total += static_cast<uint32_t>(hi[i] - lo[i]);
  }
  if (total == 0) {
    mbar_arrive(bar);
    return;
  }
  mbar_arrive_expect_tx(bar, total);
#pragma unroll
  for (int i = 0; i < kStreams; ++i)
    if (hi[i] > lo[i])
      bulk_load(slot_at + off[i], reinterpret_cast<const void*>(lo[i]), static_cast<uint32_t>(hi[i] - lo[i]), bar,
                policy);
}

// Columns of a lane: col0 + 32 e + lane, e < 8. The first out of range ends them. `full` and
// `any` are the same for the warp: only a row's last block has bounds to check.
struct OddCols {
  int col;  // of e = 0
  int n;    // how many of the eight lie in the slice
  bool full, any;  // all of the warp's, some
};

__device__ __forceinline__ OddCols odd_cols(const RowPlan& pl, const RowCtx& c, int j) {
  OddCols o;
  o.col = (j * pl.G + (c.gl & ~31)) * 8 + c.lane;
  o.n = o.col < c.ncols ? min(8, (c.ncols - o.col + 31) >> 5) : 0;
  o.full = o.col - c.lane + 256 <= c.ncols;
  o.any = o.col - c.lane < c.ncols;
  return o;
}

template <typename T, bool kFull>
__device__ __forceinline__ void odd_load(const unsigned char* p, const OddCols& o, float (&v)[8]) {
  T raw[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) raw[e] = kFull || e < o.n ? ld1(reinterpret_cast<const T*>(p) + e * 32) : T(0.f);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = static_cast<float>(raw[e]);
}

struct Any {};  // a type chosen at run time

template <typename T>
__device__ __forceinline__ void odd_read(const unsigned char* p, int dt, const OddCols& o, float (&v)[8]) {
  if constexpr (!std::is_same_v<T, Any>) {
    if (o.full) odd_load<T, true>(p, o, v); else odd_load<T, false>(p, o, v);
  } else if (dt == RMSNORM_B200_F32) {
    odd_read<float>(p, dt, o, v);
  } else if (dt == RMSNORM_B200_BF16) {
    odd_read<__nv_bfloat16>(p, dt, o, v);
  } else {
    odd_read<__half>(p, dt, o, v);
  }
}

template <typename T, bool kFull>
__device__ __forceinline__ void odd_store(void* base, int64_t at, const OddCols& o, const float (&v)[8]) {
  T* p = static_cast<T*>(base) + at;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (kFull || e < o.n) st1(p + e * 32, static_cast<T>(v[e]));
}

template <typename T>
__device__ __forceinline__ void odd_write(void* base, int dt, int64_t at, const OddCols& o, const float (&v)[8]) {
  if constexpr (!std::is_same_v<T, Any>) {
    if (o.full) odd_store<T, true>(base, at, o, v); else odd_store<T, false>(base, at, o, v);
  } else if (dt == RMSNORM_B200_F32) {
    odd_write<float>(base, dt, at, o, v);
  } else if (dt == RMSNORM_B200_BF16) {
    odd_write<__nv_bfloat16>(base, dt, at, o, v);
  } else {
    odd_write<__half>(base, dt, at, o, v);
  }
}

// weight and bias of the slice, column by column.
__device__ __forceinline__ void odd_affine(const RowPlan& pl, const RowCtx& c, const void* w, int w_dt, const void* b,
                                           int b_dt) {
  for (int i0 = threadIdx.x; i0 < c.ncols; i0 += 4 * blockDim.x) {
    float f[2][4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * static_cast<int>(blockDim.x);
      f[0][u] = w && i < c.ncols ? load1_rt(w, w_dt, c.slice0 + i) : 1.f;
      f[1][u] = pl.bias && i < c.ncols ? load1_rt(b, b_dt, c.slice0 + i) : 0.f;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * static_cast<int>(blockDim.x);
      if (i < c.ncols) c.w[i] = f[0][u];
      if (pl.bias && i < c.ncols) c.b[i] = f[1][u];
    }
  }
  __syncthreads();
}

__device__ __forceinline__ void odd_affine8(const float* a, const OddCols& o, float (&v)[8]) {
  if (o.full) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = a[o.col + e * 32];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < o.n ? a[o.col + e * 32] : 0.f;
  }
}

// Keep decisions of the lane's columns. The lane draws the words of two of the block's 64
// quads, quad `lane` and quad 32 + lane; column 32 e + lane lies in quad 8 e + lane / 4, whose
// bits come from the lane that drew it. All lanes of the warp together.
__device__ __forceinline__ uint32_t odd_keep(const DropParams& d, int64_t block_col, int64_t row, uint64_t offset,
                                             int lane) {
  const uint32_t quad = static_cast<uint32_t>(block_col >> 2) + lane, mrow = static_cast<uint32_t>(d.row0 + row);
  uint32_t a[4], b[4], mine = 0, keep = 0;
  philox(d, quad, mrow, offset, a);
  philox(d, quad + 32, mrow, offset, b);
#pragma unroll
  for (int i = 0; i < 4; ++i) mine |= (a[i] >= d.least ? 1u << i : 0u) | (b[i] >= d.least ? 16u << i : 0u);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t theirs = __shfl_sync(0xffffffffu, mine, (8 * e + (lane >> 2)) & 31);
    keep |= (theirs >> ((e & 4) + (lane & 3)) & 1u) << e;
  }
  return keep;
}

// X: type of x, the residual and a floating output; RO: of residual_out.
template <typename X, typename RO, bool kQuant, int K>
__global__ void __launch_bounds__(kOddThreads, 1) odd_fwd_kernel(const FusedFwdParams p, const RowPlan pl) {
  RowCtx c = row_begin(pl, p.N);
  pdl_launch_dependents();
  pdl_wait();
  const OddStream src[2] = {{p.x, p.x_dt, dtype_bytes(p.x_dt)}, {p.res, p.res_dt, dtype_bytes(p.res_dt)}};
  const uint64_t policy = l2_policy_evict_first();
  if (c.gl == 0)
    for (int u = 0; u < pl.S && u < c.units; ++u) odd_issue(pl, c, u, u, p.rows, p.N, src, policy);
  odd_affine(pl, c, p.w, p.w_dt, p.b, p.b_dt);
  const uint64_t offset = kQuant ? 0ull : drop_offset(p.drop);
  const float inv_n = 1.f / static_cast<float>(p.N);
  const bool i8 = p.out_dt == RMSNORM_B200_I8;
  const float inv_q = i8 ? I8::kInvQ : E4M3::kInvQ;

  int slot = 0;
  uint32_t phase = 0;
  int64_t unit = 0;
  for (int64_t tile = c.first; tile < pl.tiles; tile += c.step) {
    const int64_t row0 = tile * pl.R;
    const int nrows = static_cast<int>(min(static_cast<int64_t>(pl.R), p.rows - row0));
    for (int r = 0; r < nrows; ++r) {
      const int64_t row = row0 + r;
      const int64_t e0 = row * p.N + c.slice0;
      float h[K][8];
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < K; ++j) {
        const int first_step = j & ~(pl.KC - 1);
        if (r == 0 && j == first_step) mbar_wait_warp(&c.full[slot], phase, kSiteFwdFull);
        const OddCols o = odd_cols(pl, c, j);
        if (!o.any) {
#pragma unroll
          for (int e = 0; e < 8; ++e) h[j][e] = 0.f;
        } else {
          const unsigned char* base = c.ring + static_cast<size_t>(slot) * pl.unit_bytes;
          const int64_t first = row0 * p.N + c.slice0 + first_step * pl.G * 8;  // element of the unit
          const int at = r * static_cast<int>(p.N) + o.col - first_step * pl.G * 8;
          odd_read<X>(base + odd_lead(static_cast<const unsigned char*>(p.x) + first * src[0].bytes) + at * src[0].bytes,
                   p.x_dt, o, h[j]);
          float res[8];
          if (p.res)
            odd_read<X>(base + pl.off[1] + odd_lead(static_cast<const unsigned char*>(p.res) + first * src[1].bytes) +
                         at * src[1].bytes,
                     p.res_dt, o, res);
          if constexpr (!kQuant) {
            __syncwarp();
            const uint32_t keep = odd_keep(p.drop, c.slice0 + o.col - c.lane, row, offset, c.lane);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float v = p.res ? res[e] : 0.f;
              h[j][e] = keep >> e & 1u ? fmaf(h[j][e], p.drop.scale, v) : v;
            }
          } else if (p.res) {
#pragma unroll
            for (int e = 0; e < 8; ++e) h[j][e] += res[e];
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) ss = fmaf(h[j][e], h[j][e], ss);
          if (p.ro) odd_write<RO>(p.ro, p.ro_dt, e0 + o.col, o, h[j]);
        }
        if (r == nrows - 1 && ((j + 1) & (pl.KC - 1)) == 0) {
          if (release_unit(c, slot) && unit + pl.S < c.units)
            odd_issue(pl, c, unit + pl.S, slot, p.rows, p.N, src, policy);
          ++unit;
          if (++slot == pl.S) {
            slot = 0;
            phase ^= 1u;
          }
        }
      }
      uint32_t most = 0;
      row_total<true, false>(pl, c, ss, most, kSiteFwdCluster);
      const float rs = rsqrtf(ss * inv_n + p.eps);
      if (p.rstd && c.gl == 0 && c.rank == 0) st1(&p.rstd[row], rs);
#pragma unroll
      for (int j = 0; j < K; ++j) {
        const OddCols o = odd_cols(pl, c, j);
        if (!o.any) continue;
        float w[8], b[8];
        odd_affine8(c.w, o, w);
        if (pl.bias) odd_affine8(c.b, o, b);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          h[j][e] = h[j][e] * rs;
          h[j][e] = pl.bias ? fmaf(h[j][e], w[e], b[e]) : h[j][e] * w[e];
        }
        if (!o.full) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e >= o.n) h[j][e] = 0.f;  // rs may be NaN
        }
        if constexpr (!kQuant) odd_write<X>(p.out, p.out_dt, e0 + o.col, o, h[j]);
      }
      if constexpr (kQuant) {
        float inv_row = 0.f;
        if (p.group == 0) {
#pragma unroll
          for (int j = 0; j < K; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) most = max(most, magnitude(h[j][e]));
          float unused = 0.f;
          row_total<false, true>(pl, c, unused, most, kSiteFwdCluster);
          const float s = scale_of(__uint_as_float(most), inv_q);
          if (c.gl == 0 && c.rank == 0) st1(&p.scales[row * p.scale_row], s);
          inv_row = inverse(s);
        }
#pragma unroll
        for (int j = 0; j < K; ++j) {
          const OddCols o = odd_cols(pl, c, j);
          if (!o.any) continue;
          float inv[8];
          if (p.group) {  // 32 columns a lane step: a scale spans 1, 2, 4 or 8 of them
            uint32_t m[8];
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 8; ++e) m[e] = __reduce_max_sync(0xffffffffu, magnitude(h[j][e]));
            if (p.group >= 64)
#pragma unroll
              for (int e = 0; e < 8; e += 2) m[e] = m[e + 1] = max(m[e], m[e + 1]);
            if (p.group >= 128)
#pragma unroll
              for (int e = 0; e < 8; e += 4) m[e] = m[e + 1] = m[e + 2] = m[e + 3] = max(m[e], m[e + 2]);
            if (p.group >= 256)
#pragma unroll
              for (int e = 0; e < 8; ++e) m[e] = max(m[0], m[4]);
            float* scale = p.scales + row * p.scale_row + ((c.slice0 + o.col - c.lane) >> p.group_shift) * p.scale_group;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              if (e > 0 && (e * 32 & (p.group - 1)) != 0) {  // the scale of the step before
                inv[e] = inv[e - 1];
                continue;
              }
              const float s = scale_of(__uint_as_float(m[e]), inv_q);
              inv[e] = inverse(s);
              if (c.lane == 0 && e < o.n) st1(scale, s);
              scale += p.scale_group;
            }
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) inv[e] = inv_row;
          }
          uint8_t* dst = static_cast<uint8_t*>(p.out) + e0 + o.col;
#pragma unroll
          for (int e = 0; e < 8; ++e) h[j][e] *= inv[e];
          uint32_t q[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float2 lo = make_float2(h[j][4 * i], h[j][4 * i + 1]), hi = make_float2(h[j][4 * i + 2], h[j][4 * i + 3]);
            q[i] = i8 ? I8::pack4(lo, hi) : E4M3::pack4(lo, hi);
          }
          if (o.full) {
#pragma unroll
            for (int e = 0; e < 8; ++e) st1(dst + e * 32, static_cast<uint8_t>(q[e >> 2] >> (8 * (e & 3))));
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (e < o.n) st1(dst + e * 32, static_cast<uint8_t>(q[e >> 2] >> (8 * (e & 3))));
          }
        }
      }
    }
  }
  row_end(pl, c);
}

// H: type of h, dresidual_out and dresidual; DY: of dout and dx.
template <typename H, typename DY, int K>
__global__ void __launch_bounds__(kOddThreads, 1) odd_bwd_kernel(const FusedBwdParams p, const RowPlan pl) {
  RowCtx c = row_begin(pl, p.N);
  pdl_launch_dependents();
  pdl_wait();
  const OddStream src[3] = {{p.h, p.h_dt, dtype_bytes(p.h_dt)},
                            {p.dy, p.dy_dt, dtype_bytes(p.dy_dt)},
                            {p.dro, p.dro_dt, dtype_bytes(p.dro_dt)}};
  const uint64_t policy = l2_policy_evict_first();
  if (c.gl == 0)
    for (int u = 0; u < pl.S && u < c.units; ++u) odd_issue(pl, c, u, u, p.rows, p.N, src, policy);
  odd_affine(pl, c, p.w, p.w_dt, nullptr, 0);
  const uint64_t offset = drop_offset(p.drop);
  const float inv_n = 1.f / static_cast<float>(p.N);
  float dw[K][8], db[K][8];
#pragma unroll
  for (int j = 0; j < K; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[j][e] = db[j][e] = 0.f;

  int slot = 0;
  uint32_t phase = 0;
  int64_t unit = 0;
  for (int64_t tile = c.first; tile < pl.tiles; tile += c.step) {
    const int64_t row0 = tile * pl.R;
    const int nrows = static_cast<int>(min(static_cast<int64_t>(pl.R), p.rows - row0));
    for (int r = 0; r < nrows; ++r) {
      const int64_t row = row0 + r;
      const int64_t e0 = row * p.N + c.slice0;
      const float rs = ld1(&p.rstd[row]);
      float h[K][8], g[K][8], d[K][8];  // g becomes dy w
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < K; ++j) {
        const int first_step = j & ~(pl.KC - 1);
        if (r == 0 && j == first_step) mbar_wait_warp(&c.full[slot], phase, kSiteBwdFull);
        const OddCols o = odd_cols(pl, c, j);
        if (o.any) {
          const unsigned char* base = c.ring + static_cast<size_t>(slot) * pl.unit_bytes;
          const int64_t first = row0 * p.N + c.slice0 + first_step * pl.G * 8;
          const int at = r * static_cast<int>(p.N) + o.col - first_step * pl.G * 8;
          auto slot_of = [&](int i) {
            return base + pl.off[i] + odd_lead(static_cast<const unsigned char*>(src[i].p) + first * src[i].bytes) +
                   at * src[i].bytes;
          };
          odd_read<H>(slot_of(0), p.h_dt, o, h[j]);
          odd_read<DY>(slot_of(1), p.dy_dt, o, g[j]);
          if (p.dro) odd_read<H>(slot_of(2), p.dro_dt, o, d[j]);
          float w[8];
          odd_affine8(c.w, o, w);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float hg = h[j][e] * g[j][e];
            s = fmaf(hg, w[e], s);
            dw[j][e] = fmaf(hg, rs, dw[j][e]);
            db[j][e] += g[j][e];
            g[j][e] *= w[e];
          }
        }
        if (r == nrows - 1 && ((j + 1) & (pl.KC - 1)) == 0) {
          if (release_unit(c, slot) && unit + pl.S < c.units)
            odd_issue(pl, c, unit + pl.S, slot, p.rows, p.N, src, policy);
          ++unit;
          if (++slot == pl.S) {
            slot = 0;
            phase ^= 1u;
          }
        }
      }
      uint32_t unused = 0;
      row_total<true, false>(pl, c, s, unused, kSiteBwdCluster);
      const float t = -(s * inv_n * rs * rs * rs);  // rs^3 by itself may overflow
#pragma unroll
      for (int j = 0; j < K; ++j) {
        const OddCols o = odd_cols(pl, c, j);
        if (!o.any) continue;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = fmaf(g[j][e], rs, h[j][e] * t);
          d[j][e] = p.dro ? v + d[j][e] : v;
        }
        if (p.dres) odd_write<H>(p.dres, p.dres_dt, e0 + o.col, o, d[j]);
        __syncwarp();
        const uint32_t keep = odd_keep(p.drop, c.slice0 + o.col - c.lane, row, offset, c.lane);
#pragma unroll
        for (int e = 0; e < 8; ++e) d[j][e] = keep >> e & 1u ? d[j][e] * p.drop.scale : 0.f;
        odd_write<DY>(p.dx, p.dx_dt, e0 + o.col, o, d[j]);
      }
    }
  }
  row_end(pl, c);
  // one partial row per cluster; several groups add theirs in group order through the rings
  float* staged = reinterpret_cast<float*>(rmsb_dyn_smem);
  const int64_t part = blockIdx.x / pl.C;
  if (!p.dw_part && !p.db_part) return;
#pragma unroll
  for (int j = 0; j < K; ++j) {
    const OddCols o = odd_cols(pl, c, j);
    const int in_step = o.col - j * pl.G * 8;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      staged[(2 * c.gid) * pl.G * 8 + in_step + e * 32] = dw[j][e];
      staged[(2 * c.gid + 1) * pl.G * 8 + in_step + e * 32] = db[j][e];
    }
    __syncthreads();
    const int first = j * pl.G * 8;
    for (int i = threadIdx.x; i < pl.G * 8 && first + i < c.ncols; i += blockDim.x) {
      float v = 0.f, u = 0.f;
      for (int q = 0; q < pl.groups; ++q) {
        v += staged[(2 * q) * pl.G * 8 + i];
        u += staged[(2 * q + 1) * pl.G * 8 + i];
      }
      if (p.dw_part) st1(p.dw_part + part * p.N + c.slice0 + first + i, v);
      if (p.db_part) st1(p.db_part + part * p.N + c.slice0 + first + i, u);
    }
  }
}

}  // namespace rmsb200
