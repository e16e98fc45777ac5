// shift_bwd_kernel.cuh -- the backward of dropout + residual + RMSNorm on shifted vectors
// (shift_rows.cuh).
#pragma once

#include "fused_bwd_kernels.cuh"
#include "shift_rows.cuh"

namespace rmsb200 {

constexpr int kShiftBwdSteps = 4;  // vector steps a thread, at most: their masks are the bytes of a word

//   dh = rs dy w - h rs^3 mean(h dy w) (+ dresidual_out)
// The sums of dweight and dbias lie in tensor memory and the row is read from its slot a second
// time: neither takes registers, so the number of steps is free (the aligned kernel, which keeps
// the row in registers, has the slot reloaded sooner: 227 against 299 us at 32768 x 4096 bf16).
// H: type of h, dresidual_out and dresidual; DY: of dout and dx.
template <typename H, typename DY>
__global__ void __launch_bounds__(kShiftThreads, 1) shift_bwd_kernel(const FusedBwdParams p, const RowPlan pl) {
  constexpr int kH = sizeof(H), kDy = sizeof(DY);
  RowCtx c = row_begin(pl, p.N);
  const RowShift sh = shift_begin(pl, c, p.rows, p.N);
  pdl_launch_dependents();
  if (c.warp == 0) tmem_alloc_warp(&c.bars->tmem, kTmemCols);
  pdl_wait();
  const void* src[3] = {p.h, p.dy, p.dro};
  const int bytes[3] = {kH, kDy, p.dro ? kH : 0};
  const uint64_t policy = l2_policy_evict_first();
  if (c.gl == 0)
    for (int u = 0; u < pl.S && u < c.units; ++u) shift_issue(pl, c, sh, u, u, p.rows, p.N, src, bytes, policy);
  tmem_fence_before_sync();
  shift_affine(pl, c, sh, p.w, p.w_dt, nullptr, 0);
  tmem_fence_after_sync();
  const uint32_t tmem_base = c.bars->tmem;
  const uint32_t sums_at = tmem_base + (static_cast<uint32_t>(c.warp & 3) << 21) +
                           static_cast<uint32_t>(c.warp >> 2) * (kBwdTmemSteps * 16);
  const uint64_t offset = drop_offset(p.drop);
  const float inv_n = 1.f / static_cast<float>(p.N);
  const int width = pl.G * 8, steps = (c.ncols + width - 1) / width;  // the same for the cluster's CTA

  float2 sums[8];  // dweight, then dbias, of eight columns
#pragma unroll
  for (int i = 0; i < 8; ++i) sums[i] = make_float2(0.f, 0.f);
  for (int j = 0; j < steps; ++j) tmem_st16(sums_at + j * 16, sums);

  int slot = 0;
  uint32_t phase = 0;
  int64_t unit = 0;
  float rs_next = c.units > 0 ? ld1(&p.rstd[c.first]) : 0.f;  // a row ahead of its use
  for (int64_t row = c.first; row < p.rows; row += c.step) {
    const int64_t e0 = row * p.N - sh.lead + c.slice0;
    const float rs = rs_next;
    if (row + c.step < p.rows) rs_next = ld1(&p.rstd[row + c.step]);
    const unsigned char* base = c.ring + static_cast<size_t>(slot) * pl.unit_bytes;
    mbar_wait_warp(&c.full[slot], phase, kSiteBwdFull);
    float2 s2 = make_float2(0.f, 0.f);
    for (int j = 0; j < steps; ++j) {
      const int col = j * width + c.gl * 8;
      if (col >= c.ncols) break;
      float2 h[4], g[4], w[4];
      Pair8<H>::load(base + col * kH, h);
      Pair8<DY>::load(base + pl.off[1] + col * kDy, g);
      const ShiftEdge edge(sh, c.slice0 + col);
      if (!edge.whole()) {
        edge.mask(h);
        edge.mask(g);
      }
      affine8(pl, c.w, col, w);
#pragma unroll
      for (int i = 0; i < 4; ++i) s2 = fma2(mul2(h[i], g[i]), w[i], s2);
    }
    __syncwarp();
    float s = s2.x + s2.y;
    uint32_t unused = 0, keep = 0;  // the masks, drawn while the row's total comes together
    row_total<true, false>(pl, c, s, unused, kSiteBwdCluster, [&] {
      __syncwarp();
      keep = shift_keep<kShiftBwdSteps>(p.drop, pl, c, sh, row, offset);
    });
    const float t = -(s * inv_n * rs * rs * rs);  // rs^3 by itself may overflow
    tmem_wait_st();  // of the row before
    for (int j = 0; j < steps; ++j) {
      const int col = j * width + c.gl * 8;
      __syncwarp();
      tmem_ld16(sums_at + j * 16, sums);
      float2 d[4], g[4], w[4];
      const ShiftEdge edge(sh, c.slice0 + col);
      if (col < c.ncols) {
        Pair8<H>::load(base + col * kH, d);
        Pair8<DY>::load(base + pl.off[1] + col * kDy, g);
        if (!edge.whole()) {
          edge.mask(d);
          edge.mask(g);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = g[i] = make_float2(0.f, 0.f);
      }
      __syncwarp();
      tmem_wait_ld();
      add_sums(sums, d, g, rs);
      tmem_st16(sums_at + j * 16, sums);
      if (col >= c.ncols) continue;
      affine8(pl, c.w, col, w);
#pragma unroll
      for (int i = 0; i < 4; ++i) d[i] = fma2(g[i], w[i], mul2(d[i], splat2(t)));
      if (p.dro) {
        Pair8<H>::load(base + pl.off[2] + col * kH, g);
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = add2(d[i], g[i]);
      }
      if (p.dres) shift_store<H>(p.dres, e0 + col, edge, d);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        g[i] = mul2(d[i], splat2(p.drop.scale));
        if (!(keep >> (8 * j + 2 * i) & 1u)) g[i].x = 0.f;
        if (!(keep >> (8 * j + 2 * i + 1) & 1u)) g[i].y = 0.f;
      }
      shift_store<DY>(p.dx, e0 + col, edge, g);
    }
    if (release_unit(c, slot) && unit + pl.S < c.units)
      shift_issue(pl, c, sh, unit + pl.S, slot, p.rows, p.N, src, bytes, policy);
    __syncwarp();
    ++unit;
    if (++slot == pl.S) {
      slot = 0;
      phase ^= 1u;
    }
  }
  row_end(pl, c);
  __syncwarp();
  // One partial row of dweight and of dbias per cluster. The groups add theirs in group order
  // through the rings, whose every copy has landed and been read.
  tmem_wait_st();
  float* staged = reinterpret_cast<float*>(rmsb_dyn_smem);
  const int64_t part = blockIdx.x / pl.C;
  const bool want = p.dw_part || p.db_part;
  for (int j = 0; want && j < steps; ++j) {
    __syncwarp();
    tmem_ld16(sums_at + j * 16, sums);
    tmem_wait_ld();
    __syncthreads();
    float2* q = reinterpret_cast<float2*>(staged + (2 * c.gid) * width + c.gl * 8);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      q[i] = sums[i];
      q[pl.G * 4 + i] = sums[4 + i];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < width && j * width + i < c.ncols; i += blockDim.x) {
      const int64_t n = c.slice0 + j * width + i - sh.lead;
      if (n < 0) continue;
      float v = 0.f, u = 0.f;
      for (int g = 0; g < pl.groups; ++g) {
        v += staged[(2 * g) * width + i];
        u += staged[(2 * g + 1) * width + i];
      }
      if (p.dw_part) st1(p.dw_part + part * p.N + n, v);
      if (p.db_part) st1(p.db_part + part * p.N + n, u);
    }
  }
  tmem_fence_before_sync();
  __syncthreads();
  tmem_fence_after_sync();
  if (c.warp == 0) tmem_dealloc_warp(tmem_base, kTmemCols);
}

}  // namespace rmsb200
