// shift_fwd_kernel.cuh -- the forward of the fused row operators on shifted vectors (shift_rows.cuh).
#pragma once

#include "fused_fwd_kernels.cuh"
#include "shift_rows.cuh"

namespace rmsb200 {

constexpr int kShiftFwdSteps = 4;  // vector steps a thread, or one

// X: type of x and of a floating output; residual and residual_out have it too, or fp32, or are
// absent. 8-bit outputs have a scale a row.
template <typename X, typename End, int K>
__global__ void __launch_bounds__(kShiftThreads, 1) shift_fwd_kernel(const FusedFwdParams p, const RowPlan pl) {
  constexpr bool kQuant = End::kQuant;
  constexpr int kX = sizeof(X);
  RowCtx c = row_begin(pl, p.N);
  const RowShift sh = shift_begin(pl, c, p.rows, p.N);
  pdl_launch_dependents();
  pdl_wait();
  const bool res_f32 = p.res_dt == RMSNORM_B200_F32, ro_f32 = p.ro_dt == RMSNORM_B200_F32;
  const int res_bytes = p.res ? (res_f32 ? 4 : kX) : 0;
  const void* src[2] = {p.x, p.res};
  const int bytes[2] = {kX, res_bytes};
  const uint64_t policy = l2_policy_evict_first();
  if (c.gl == 0)
    for (int u = 0; u < pl.S && u < c.units; ++u) shift_issue(pl, c, sh, u, u, p.rows, p.N, src, bytes, policy);
  shift_affine(pl, c, sh, p.w, p.w_dt, p.b, p.b_dt);
  const uint64_t offset = kQuant ? 0ull : drop_offset(p.drop);
  const float inv_n = 1.f / static_cast<float>(p.N);

  int slot = 0;
  uint32_t phase = 0;
  int64_t unit = 0;
  for (int64_t row = c.first; row < p.rows; row += c.step) {
    const int64_t e0 = row * p.N - sh.lead + c.slice0;
    float2 h[K][4];
    float2 ss = make_float2(0.f, 0.f);
    uint32_t keep = 0;
    if constexpr (!kQuant) keep = shift_keep<K>(p.drop, pl, c, sh, row, offset);
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int first_step = j & ~(pl.KC - 1);
      if (j == first_step) mbar_wait(&c.full[slot], phase, kSiteFwdFull);
      const int col = (j * pl.G + c.gl) * 8;
      if (col < c.ncols) {
        const unsigned char* base = c.ring + static_cast<size_t>(slot) * pl.unit_bytes;
        const int at = col - first_step * pl.G * 8;
        const ShiftEdge edge(sh, c.slice0 + col);
        Pair8<X>::load(base + at * kX, h[j]);
        float2 res[4];
#pragma unroll
        for (float2& v : res) v = make_float2(0.f, 0.f);
        if (p.res) shift_load<X>(base + pl.off[1] + at * res_bytes, res_f32, res);
        if constexpr (!kQuant) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 kept = fma2(h[j][i], splat2(p.drop.scale), res[i]);
            h[j][i].x = keep >> (8 * j + 2 * i) & 1u ? kept.x : res[i].x;
            h[j][i].y = keep >> (8 * j + 2 * i + 1) & 1u ? kept.y : res[i].y;
          }
        } else if (p.res) {
#pragma unroll
          for (int i = 0; i < 4; ++i) h[j][i] = add2(h[j][i], res[i]);
        }
        if (!edge.whole()) edge.mask(h[j]);
#pragma unroll
        for (int i = 0; i < 4; ++i) ss = fma2(h[j][i], h[j][i], ss);
        if (p.ro) {
          if (ro_f32)
            shift_store<float>(p.ro, e0 + col, edge, h[j]);
          else
            shift_store<X>(p.ro, e0 + col, edge, h[j]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) h[j][i] = make_float2(0.f, 0.f);
      }
      if (((j + 1) & (pl.KC - 1)) == 0) {
        if (release_unit(c, slot) && unit + pl.S < c.units)
          shift_issue(pl, c, sh, unit + pl.S, slot, p.rows, p.N, src, bytes, policy);
        ++unit;
        if (++slot == pl.S) {
          slot = 0;
          phase ^= 1u;
        }
      }
    }
    float sum = ss.x + ss.y;
    uint32_t bits = 0;
    row_total<true, false>(pl, c, sum, bits, kSiteFwdCluster);
    const float rs = rsqrtf(sum * inv_n + p.eps);
    if (p.rstd && c.gl == 0 && c.rank == 0) st1(&p.rstd[row], rs);
    float most = 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j) {  // y in the place of h
      const int col = (j * pl.G + c.gl) * 8;
      if (col >= c.ncols) continue;
      const ShiftEdge edge(sh, c.slice0 + col);
      float2 w[4], b[4];
      affine8(pl, c.w, col, w);
#pragma unroll
      for (float2& v : b) v = make_float2(0.f, 0.f);
      if (pl.bias) affine8(pl, c.b, col, b);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 y = mul2(h[j][i], splat2(rs));
        h[j][i] = pl.bias ? fma2(y, w[i], b[i]) : mul2(y, w[i]);
      }
      if constexpr (kQuant) {
        if (!edge.whole()) edge.mask(h[j]);  // rs may be NaN
        most = largest8(most, h[j]);
      } else {
        shift_store<X>(p.out, e0 + col, edge, h[j]);
      }
    }
    if constexpr (kQuant) {
      using Q = typename End::Type;
      bits = magnitude(most);
      float unused = 0.f;
      row_total<false, true>(pl, c, unused, bits, kSiteFwdCluster);
      const float s = scale_of(__uint_as_float(bits), Q::kInvQ), inv = inverse(s);
      if (c.gl == 0 && c.rank == 0) st1(&p.scales[row * p.scale_row], s);
#pragma unroll
      for (int j = 0; j < K; ++j) {
        const int col = (j * pl.G + c.gl) * 8;
        if (col >= c.ncols) continue;
        const ShiftEdge edge(sh, c.slice0 + col);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[j][i] = mul2(h[j][i], splat2(inv));
        const uint32_t q[2] = {Q::pack4(h[j][0], h[j][1]), Q::pack4(h[j][2], h[j][3])};
        uint8_t* dst = static_cast<uint8_t*>(p.out) + e0 + col;
        if (edge.whole()) {
          if (RMSB_DBG_OK(dst, 8, kDbgVecStore)) __stcs(reinterpret_cast<uint2*>(dst), make_uint2(q[0], q[1]));
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (i >= edge.lo && i < edge.hi) st1(dst + i, static_cast<uint8_t>(q[i >> 2] >> (8 * (i & 3))));
        }
      }
    }
  }
  row_end(pl, c);
}

}  // namespace rmsb200
