// shift_fwd_kernel.cuh -- the forward of the fused row operators on shifted vectors (shift_rows.cuh).
#pragma once

#include "fused_fwd_kernels.cuh"
#include "shift_rows.cuh"

namespace rmsb200 {

constexpr int kShiftFwdSteps = 4;  // vector steps a thread, or one

// X: type of x and of a floating output; residual and residual_out have it too, or fp32, or are
// absent.
// A scale's columns begin `lead` elements into a vector, so the largest values of the groups are
// put together in shared memory: a group's lanes are neighbours, their first lane adds the
// maximum of its own elements and, of the elements before them, to the group before.
// Maxima do not depend on their order. Two sets take turns; a row's is cleared after the
// total of the row after it, which every warp reaches when it has read the scales.
template <typename X, typename End, int K>
__global__ void __launch_bounds__(kShiftThreads, 1) shift_fwd_kernel(const FusedFwdParams p, const RowPlan pl) {
  constexpr bool kQuant = End::kQuant, kGroups = kQuant && !End::kRowScale;
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
  uint32_t* largest = reinterpret_cast<uint32_t*>(c.bars + 1) + c.gid * 2 * pl.scale_slots;  // of this row; then of the row before
  uint32_t* cleared = largest + pl.scale_slots;
  if constexpr (kGroups)
    for (int i = c.gl; i < 2 * pl.scale_slots; i += pl.G) largest[i] = 0;
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
      if (j == first_step) mbar_wait_warp(&c.full[slot], phase, kSiteFwdFull);
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
        if constexpr (!kGroups) most = largest8(most, h[j]);
      } else {
        shift_store<X>(p.out, e0 + col, edge, h[j]);
      }
    }
    if constexpr (kQuant) {
      using Q = typename End::Type;
      float inv_row = 0.f;
      float unused = 0.f;
      bits = magnitude(most);
      if constexpr (kGroups) {
#pragma unroll
        for (int j = 0; j < K; ++j) {
          const int col = (j * pl.G + c.gl) * 8;
          const bool first = (col & (p.group - 1)) == 0;
          const int own = first ? sh.lead : 0;  // elements from there on are this group's
          uint32_t here = 0, before = 0;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t m = magnitude(i & 1 ? h[j][i >> 1].y : h[j][i >> 1].x);
            if (i >= own)
              here = max(here, m);
            else
              before = max(before, m);
          }
          for (int o = p.group >> 4; o > 0; o >>= 1) here = max(here, __shfl_xor_sync(0xffffffffu, here, o));
          if (first && col < c.ncols) {
            atomicMax(&largest[col >> p.group_shift], here);
            if (own > 0 && col > 0) atomicMax(&largest[(col >> p.group_shift) - 1], before);
          }
        }
        __syncwarp();
        row_total<false, true>(pl, c, unused, bits, kSiteFwdCluster);
        __syncwarp();
        for (int i = c.gl; i < pl.scale_slots; i += pl.G) cleared[i] = 0;
      } else {
        row_total<false, true>(pl, c, unused, bits, kSiteFwdCluster);
        const float s = scale_of(__uint_as_float(bits), Q::kInvQ);
        inv_row = inverse(s);
        if (c.gl == 0 && c.rank == 0) st1(&p.scales[row * p.scale_row], s);
      }
#pragma unroll
      for (int j = 0; j < K; ++j) {
        const int col = (j * pl.G + c.gl) * 8;
        if (col >= c.ncols) continue;
        const ShiftEdge edge(sh, c.slice0 + col);
        if constexpr (kGroups) {
          const int g = col >> p.group_shift;
          const bool first = (col & (p.group - 1)) == 0;
          const float s = scale_of(__uint_as_float(largest[g]), Q::kInvQ);
          const float inv = inverse(s);
          const float inv_before =
              first && g > 0 ? inverse(scale_of(__uint_as_float(largest[g - 1]), Q::kInvQ)) : inv;
          if (first && col < p.N) st1(&p.scales[row * p.scale_row + g * p.scale_group], s);
          const int own = first ? sh.lead : 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            h[j][i].x *= 2 * i >= own ? inv : inv_before;
            h[j][i].y *= 2 * i + 1 >= own ? inv : inv_before;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) h[j][i] = mul2(h[j][i], splat2(inv_row));
        }
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
      uint32_t* last = largest;
      largest = cleared;
      cleared = last;
    }
  }
  row_end(pl, c);
}

}  // namespace rmsb200
