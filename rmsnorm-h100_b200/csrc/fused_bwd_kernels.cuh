// fused_bwd_kernels.cuh -- the streaming backward of dropout + residual + RMSNorm.
#pragma once

#include "fused_generic.cuh"
#include "row_ring.cuh"

namespace rmsb200 {

constexpr int kBwdThreads = 512;
constexpr int kBwdRegSteps = 2;    // vector steps a thread whose sums stay in registers
constexpr int kBwdTmemSteps = 4;   // in tensor memory
constexpr uint32_t kTmemCols = 256;

// One vector of a tensor as loaded: 4 registers, 8 for fp32. A row is held like this from the
// first pass to the second, so its slot loads again in between.
template <typename T>
struct Raw8 {
  static constexpr int kWords = Vec8<T>::kBytes / 16;
  uint4 v[kWords];
  __device__ __forceinline__ void load(const void* p) {
#pragma unroll
    for (int i = 0; i < kWords; ++i)
      v[i] = RMSB_DBG_OK(static_cast<const uint4*>(p) + i, 16, kDbgVecLoad) ? static_cast<const uint4*>(p)[i]
                                                                          : make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) v[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void get(float2 (&f)[4]) const {
    if constexpr (kWords == 2) {
      f[0] = make_float2(__uint_as_float(v[0].x), __uint_as_float(v[0].y));
      f[1] = make_float2(__uint_as_float(v[0].z), __uint_as_float(v[0].w));
      f[2] = make_float2(__uint_as_float(v[1].x), __uint_as_float(v[1].y));
      f[3] = make_float2(__uint_as_float(v[1].z), __uint_as_float(v[1].w));
    } else {
      Pair8<T>::unpack(v[0], f);
    }
  }
};

// A vector's contribution to its columns' sums: dweight, then dbias. g becomes dy rs.
__device__ __forceinline__ void add_sums(float2 (&sum)[8], const float2 (&h)[4], float2 (&g)[4], float rs) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    sum[4 + i] = add2(g[i], sum[4 + i]);
    g[i] = mul2(g[i], splat2(rs));
    sum[i] = fma2(h[i], g[i], sum[i]);
  }
}

// H: type of h (and of dresidual), DY: of dout (and of dx), DRO: of dresidual_out, DRES: of
// dresidual (NoT: absent).
//   dh = rs dy w - h rs^3 mean(h dy w) (+ dresidual_out)
// What a warp does once a row (waits, releases, the total) costs as much as a vector step, so
// four steps a thread pay, for 16-bit rows at least. dweight and dbias are summed over a
// thread's rows: 16 registers a step, which with four steps leave no room for the row itself.
// They are kept in tensor memory then, which this kernel has no other use for: 16 columns of
// the thread's lane a step, read and written once a row. Those kernels have the row group's
// size kG built in (0: chosen at run time).
// Measured: bf16 throughout, 32768 x 16384 990 to 1000 us (820 us of bytes at a copy's rate; bound
// by instructions, 304 for eight columns, 80 of them the generator's and 16 the choice by its
// words, issued at half the SM's rate by 16 warps); 1.3e8 elements at 1024, 4096 and 8192 columns
// 217, 227 and 236 us (205 us of bytes); fp32 h, 4096 columns 359 us (328 us).
template <typename H, typename DY, typename DRO, typename DRES, int K, int kG>
__global__ void __launch_bounds__(kBwdThreads, 1) fused_bwd_kernel(const FusedBwdParams p, const RowPlan pl) {
  constexpr bool kDro = Present<DRO>::value, kDres = Present<DRES>::value, kTmem = K > kBwdRegSteps;
  constexpr int kStreams = kDro ? 3 : 2;
  constexpr int kH = Vec8<H>::kBytes / 8, kDy = Vec8<DY>::kBytes / 8;
  RowCtx c = row_begin(pl, p.N);
  const int G = kTmem ? kG : pl.G, KC = kTmem ? bwd_unit_steps(kG) : pl.KC, R = kTmem ? 1 : pl.R;
  if constexpr (kTmem) {
    if (c.warp == 0) {
      tmem_alloc_warp(&c.bars->tmem, kTmemCols);
      pdl_launch_dependents();  // for the CTA, and not before: they may take tensor memory and wait for this grid
    }
  } else {
    pdl_launch_dependents();
  }
  pdl_wait();
  const void* src[kStreams];
  int bytes[kStreams];
  src[0] = p.h;
  bytes[0] = kH;
  src[1] = p.dy;
  bytes[1] = kDy;
  if constexpr (kDro) {
    src[2] = p.dro;
    bytes[2] = Vec8<DRO>::kBytes / 8;
  }
  const uint64_t policy = l2_policy_evict_first();
  if (c.gl == 0)
    for (int u = 0; u < pl.S && u < c.units; ++u) issue_unit(pl, c, u, u, p.rows, p.N, src, bytes, policy);
  if constexpr (kTmem) tmem_fence_before_sync();
  load_affine(pl, c, p.w, p.w_dt, nullptr, 0);
  uint32_t tmem_base = 0, sums_at = 0;  // a warp reaches the 32 lanes of its quarter: the warps of a quarter side by side
  if constexpr (kTmem) {
    tmem_fence_after_sync();
    tmem_base = c.bars->tmem;
    sums_at = tmem_base + (static_cast<uint32_t>(c.warp & 3) << 21) + static_cast<uint32_t>(c.warp >> 2) * (K * 16);
  }
  const uint64_t offset = drop_offset(p.drop);
  const float inv_n = 1.f / static_cast<float>(p.N);

  float2 sums[kTmem ? 1 : K][8];  // dweight, then dbias, of eight columns
#pragma unroll
  for (int j = 0; j < (kTmem ? 1 : K); ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) sums[j][i] = make_float2(0.f, 0.f);
  if constexpr (kTmem) {
#pragma unroll
    for (int j = 0; j < K; ++j) tmem_st16(sums_at + j * 16, sums[0]);
  }

  int slot = 0;
  uint32_t phase = 0;
  int64_t unit = 0;
  float rs_next = c.units > 0 ? ld1(&p.rstd[c.first * R]) : 0.f;  // a row ahead of its use
  for (int64_t tile = c.first; tile < pl.tiles; tile += c.step) {
    const int64_t row0 = tile * R;
    const int nrows = kTmem ? 1 : static_cast<int>(min(static_cast<int64_t>(R), p.rows - row0));
    for (int r = 0; r < nrows; ++r) {
      const int64_t row = row0 + r;
      const int64_t e0 = row * p.N + c.slice0;
      const float rs = rs_next;
      const int64_t next = r + 1 < nrows ? row + 1 : (tile + c.step) * R;
      if (next < p.rows) rs_next = ld1(&p.rstd[next]);
      Raw8<H> h[K];
      Raw8<DY> dy[K];
      Raw8<std::conditional_t<kDro, DRO, __half>> dro[kDro ? K : 1];
      float2 s2 = make_float2(0.f, 0.f);
#pragma unroll
      for (int j = 0; j < K; ++j) {
        const int first_step = j & ~(KC - 1);
        const int col = j * (G * 8) + c.gl * 8;
        if (r == 0 && j == first_step) mbar_wait_warp(&c.full[slot], phase, kSiteBwdFull);
        if (col < c.ncols) {
          const unsigned char* base = c.ring + static_cast<size_t>(slot) * pl.unit_bytes;
          const int at = (kTmem ? 0 : r * static_cast<int>(p.N)) + c.gl * 8 + (j - first_step) * (G * 8);
          h[j].load(base + at * kH);
          dy[j].load(base + pl.off[1] + at * kDy);
          if constexpr (kDro) dro[j].load(base + pl.off[2] + at * (Vec8<DRO>::kBytes / 8));
          float2 hv[4], g[4], w[4];
          h[j].get(hv);
          dy[j].get(g);
          affine8(pl, c.w, col, w);
#pragma unroll
          for (int i = 0; i < 4; ++i) s2 = fma2(mul2(hv[i], g[i]), w[i], s2);
          if constexpr (!kTmem) add_sums(sums[j], hv, g, rs);
        } else {
          h[j].zero();
          dy[j].zero();
        }
        if (r == nrows - 1 && ((j + 1) & (KC - 1)) == 0) {
          if (release_unit(c, slot) && unit + pl.S < c.units)
            issue_unit(pl, c, unit + pl.S, slot, p.rows, p.N, src, bytes, policy);
          __syncwarp();
          ++unit;
          if (++slot == pl.S) {
            slot = 0;
            phase ^= 1u;
          }
        }
      }
      float s = s2.x + s2.y;
      uint32_t unused = 0;
      // the first step's mask is drawn while the row's total comes together
      uint32_t words[2][4];
      row_total<true, false>(pl, c, s, unused, kSiteBwdCluster,
                             [&] { draw8(p.drop, c.slice0 + c.gl * 8, row, offset, words); });
      const float t = -(s * inv_n * rs * rs * rs);  // rs^3 by itself may overflow
      if constexpr (kTmem) tmem_wait_st();  // of the row before
#pragma unroll
      for (int j = 0; j < K; ++j) {
        const int col = j * (G * 8) + c.gl * 8;
        // tensor memory is slow to answer: asked before the mask is drawn, read after it
        if constexpr (kTmem) {
          __syncwarp();
          tmem_ld16(sums_at + j * 16, sums[0]);
        } else if (col >= c.ncols) {
          continue;
        }
        if (j > 0) draw8(p.drop, c.slice0 + col, row, offset, words);
        float2 d[4], g[4], w[4];
        h[j].get(d);
        dy[j].get(g);
        if constexpr (kTmem) {
          tmem_wait_ld();
          add_sums(sums[0], d, g, rs);
          tmem_st16(sums_at + j * 16, sums[0]);
          if (col >= c.ncols) continue;
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) g[i] = mul2(g[i], splat2(rs));
        }
        affine8(pl, c.w, col, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = fma2(g[i], w[i], mul2(d[i], splat2(t)));
        if constexpr (kDro) {
          dro[j].get(g);
#pragma unroll
          for (int i = 0; i < 4; ++i) d[i] = add2(d[i], g[i]);
        }
        if constexpr (kDres)
          Pair8<DRES>::store(static_cast<unsigned char*>(p.dres) + (e0 + col) * (Vec8<DRES>::kBytes / 8), d);
        float2 zero[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          d[i] = mul2(d[i], splat2(p.drop.scale));
          zero[i] = make_float2(0.f, 0.f);
        }
        select8(p.drop, words, d, zero, g);
        Pair8<DY>::store(static_cast<unsigned char*>(p.dx) + (e0 + col) * kDy, g);
      }
      if constexpr (kTmem) __syncwarp();  // together again for the next row's tensor memory accesses
    }
  }
  row_end(pl, c);
  __syncwarp();
  // One partial row of dweight and of dbias per cluster. Several groups add theirs in group
  // order through the rings, whose every copy has landed and been read.
  if constexpr (kTmem) tmem_wait_st();
  float* staged = reinterpret_cast<float*>(rmsb_dyn_smem);
  const int64_t part = blockIdx.x / pl.C;
  const bool want = p.dw_part || p.db_part;
#pragma unroll
  for (int j = 0; j < K; ++j) {
    if (!want) break;
    const int col = (j * pl.G + c.gl) * 8;
    float2(&sum)[8] = sums[kTmem ? 0 : j];
    if constexpr (kTmem) {
      __syncwarp();
      tmem_ld16(sums_at + j * 16, sum);
      tmem_wait_ld();
    }
    const float2 dw[4] = {sum[0], sum[1], sum[2], sum[3]}, db[4] = {sum[4], sum[5], sum[6], sum[7]};
    if (pl.groups == 1) {
      if (col < c.ncols) {
        float* dst = p.dw_part + part * p.N + c.slice0 + col;
        if (p.dw_part) Pair8<float>::store(dst, dw);
        dst = p.db_part + part * p.N + c.slice0 + col;
        if (p.db_part) Pair8<float>::store(dst, db);
      }
      continue;
    }
    __syncthreads();
    if (col < c.ncols) {
      float2* q = reinterpret_cast<float2*>(staged + (2 * c.gid) * pl.G * 8 + c.gl * 8);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        q[i] = dw[i];
        q[pl.G * 4 + i] = db[i];
      }
    }
    __syncthreads();
    const int first = j * pl.G * 8;  // columns of this step
    for (int i = threadIdx.x; i < pl.G * 8 && first + i < c.ncols; i += blockDim.x) {
      float v = 0.f, u = 0.f;
      for (int g = 0; g < pl.groups; ++g) {
        v += staged[(2 * g) * pl.G * 8 + i];
        u += staged[(2 * g + 1) * pl.G * 8 + i];
      }
      if (p.dw_part) st1(p.dw_part + part * p.N + c.slice0 + first + i, v);
      if (p.db_part) st1(p.db_part + part * p.N + c.slice0 + first + i, u);
    }
  }
  if constexpr (kTmem) {
    tmem_fence_before_sync();
    __syncthreads();
    tmem_fence_after_sync();
    if (c.warp == 0) tmem_dealloc_warp(tmem_base, kTmemCols);
  }
}

// The scalar kernel: one CTA per row, types chosen at run time, the row read again from cache.
// dx and dresidual; dweight and dbias are column sums of their own (bwd_generic_partials_kernel).
__global__ void __launch_bounds__(kGenericThreads) fused_bwd_generic_kernel(const FusedBwdParams p) {
  __shared__ float red[32];
  pdl_wait();
  const uint64_t offset = drop_offset(p.drop);
  const int64_t N = p.N;
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const float rs = ld1(&p.rstd[r]);
    auto wdy = [&](int64_t n) {
      const float w = p.w ? load1_rt(p.w, p.w_dt, n) : 1.f;
      return load1_rt(p.dy, p.dy_dt, r * N + n) * w;
    };
    float c = 0.f;
    for (int64_t n = threadIdx.x; n < N; n += blockDim.x) c = fmaf(load1_rt(p.h, p.h_dt, r * N + n) * rs, wdy(n), c);
    c = block_sum_fixed(c, red) / static_cast<float>(N);
    for (int64_t n = threadIdx.x; n < N; n += blockDim.x) {
      const int64_t e = r * N + n;
      float d = (wdy(n) - load1_rt(p.h, p.h_dt, e) * rs * c) * rs;
      if (p.dro) d += load1_rt(p.dro, p.dro_dt, e);
      if (p.dres) store1_rt(p.dres, p.dres_dt, e, d);
      store1_rt(p.dx, p.dx_dt, e, keep1(p.drop, n, r, offset) ? d * p.drop.scale : 0.f);
    }
  }
}

}  // namespace rmsb200
