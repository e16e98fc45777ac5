// fused_bwd_kernels.cuh -- the streaming backward of dropout + residual + RMSNorm.
#pragma once

#include "fused_generic.cuh"
#include "row_ring.cuh"

namespace rmsb200 {

constexpr int kBwdSteps = 2;  // vector steps a thread: its dweight and dbias sums take 16 registers each

// One row's values of one tensor as loaded: 4 registers a vector, 8 for fp32.
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
  __device__ __forceinline__ void get(float (&f)[8]) const {
    if constexpr (kWords == 2) {
      f[0] = __uint_as_float(v[0].x); f[1] = __uint_as_float(v[0].y);
      f[2] = __uint_as_float(v[0].z); f[3] = __uint_as_float(v[0].w);
      f[4] = __uint_as_float(v[1].x); f[5] = __uint_as_float(v[1].y);
      f[6] = __uint_as_float(v[1].z); f[7] = __uint_as_float(v[1].w);
    } else {
      Vec8<T>::unpack(v[0], f);
    }
  }
};

// H: type of h, DY: of dout, DRO: of dresidual_out (NoT without one).
template <typename H, typename DY, typename DRO, int K>
__global__ void __launch_bounds__(kRowThreads, 1) fused_bwd_kernel(const FusedBwdParams p, const RowPlan pl) {
  constexpr bool kDro = Present<DRO>::value;
  constexpr int kStreams = kDro ? 3 : 2;
  RowCtx c = row_begin(pl, p.N);
  pdl_launch_dependents();
  pdl_wait();
  const void* src[kStreams];
  int bytes[kStreams];
  src[0] = p.h;
  bytes[0] = Vec8<H>::kBytes / 8;
  src[1] = p.dy;
  bytes[1] = Vec8<DY>::kBytes / 8;
  if constexpr (kDro) {
    src[2] = p.dro;
    bytes[2] = Vec8<DRO>::kBytes / 8;
  }
  const uint64_t policy = l2_policy_evict_first();
  if (c.gl == 0)
    for (int u = 0; u < pl.S && u < c.units; ++u) issue_unit(pl, c, u, u, p.rows, p.N, src, bytes, policy);
  load_affine(pl, c, p.w, p.w_dt, nullptr, 0);
  const uint64_t offset = drop_offset(p.drop);
  const float inv_n = 1.f / static_cast<float>(p.N);

  float dw[K][8], db[K][8];
#pragma unroll
  for (int j = 0; j < K; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[j][i] = db[j][i] = 0.f;

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
      Raw8<H> h[K];
      Raw8<DY> dy[K];
      Raw8<std::conditional_t<kDro, DRO, __half>> dro[kDro ? K : 1];
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < K; ++j) {
        const int first_step = j & ~(pl.KC - 1);
        if (r == 0 && j == first_step) mbar_wait(&c.full[slot], phase, kSiteBwdFull);
        const int col = (j * pl.G + c.gl) * 8;
        if (col < c.ncols) {
          const unsigned char* base = c.ring + static_cast<size_t>(slot) * pl.unit_bytes;
          const int at = r * static_cast<int>(p.N) + col - first_step * pl.G * 8;
          h[j].load(base + at * (Vec8<H>::kBytes / 8));
          dy[j].load(base + pl.off[1] + at * (Vec8<DY>::kBytes / 8));
          if constexpr (kDro) dro[j].load(base + pl.off[2] + at * (Vec8<DRO>::kBytes / 8));
          float hv[8], g[8], w[8];
          h[j].get(hv);
          dy[j].get(g);
          lds8(c.w + col, w);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float hg = hv[i] * g[i];
            s = fmaf(hg, w[i], s);
            dw[j][i] = fmaf(hg, rs, dw[j][i]);
            db[j][i] += g[i];
          }
        }
        if (r == nrows - 1 && ((j + 1) & (pl.KC - 1)) == 0) {
          if (release_unit(c, slot) && unit + pl.S < c.units)
            issue_unit(pl, c, unit + pl.S, slot, p.rows, p.N, src, bytes, policy);
          ++unit;
          if (++slot == pl.S) {
            slot = 0;
            phase ^= 1u;
          }
        }
      }
      uint32_t unused = 0;
      row_total<true, false>(pl, c, s, unused, kSiteBwdCluster);
      const float t = rs * rs * rs * (s * inv_n);  // dh = rs dy w - h rs^3 mean(h dy w)
#pragma unroll
      for (int j = 0; j < K; ++j) {
        const int col = (j * pl.G + c.gl) * 8;
        if (col >= c.ncols) continue;
        float hv[8], g[8], w[8], d[8];
        h[j].get(hv);
        dy[j].get(g);
        lds8(c.w + col, w);
        if constexpr (kDro) {
          dro[j].get(d);
#pragma unroll
          for (int i = 0; i < 8; ++i) d[i] += fmaf(-hv[i], t, g[i] * w[i] * rs);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) d[i] = fmaf(-hv[i], t, g[i] * w[i] * rs);
        }
        if (p.dres) store8_rt(p.dres, p.dres_dt, e0 + col, d);
        const uint32_t keep = keep8(p.drop, c.slice0 + col, row, offset);
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = keep >> i & 1u ? d[i] * p.drop.scale : 0.f;
        store8_rt(p.dx, p.dx_dt, e0 + col, d);
      }
    }
  }
  row_end(pl, c);
  // The groups' sums, one partial row per cluster: through the rings (every copy has landed
  // and been read), added in group order.
  if (!p.dw_part && !p.db_part) return;
  float* sums = reinterpret_cast<float*>(rmsb_dyn_smem);
  const int64_t part = blockIdx.x / pl.C;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float* out = which == 0 ? p.dw_part : p.db_part;
    if (!out) continue;
    float* dst = out + part * p.N + c.slice0;
    if (pl.groups == 1) {
#pragma unroll
      for (int j = 0; j < K; ++j) {
        const int col = (j * pl.G + c.gl) * 8;
        if (col < c.ncols) Vec8<float>::store(dst + col, which == 0 ? dw[j] : db[j]);
      }
      continue;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int col = (j * pl.G + c.gl) * 8;
      if (col < c.ncols) {
        float* q = sums + c.gid * pl.slice + col;
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = which == 0 ? dw[j][i] : db[j][i];
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < c.ncols; i += blockDim.x) {
      float v = 0.f;
      for (int g = 0; g < pl.groups; ++g) v += sums[g * pl.slice + i];
      st1(&dst[i], v);
    }
  }
}

}  // namespace rmsb200
