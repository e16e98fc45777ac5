// fused_fwd_kernels.cuh -- the streaming forward of the fused row operators.
#pragma once

#include "fused_generic.cuh"
#include "row_ring.cuh"

namespace rmsb200 {

// RT is NoT without a residual. kDrop: dropout, floating output; otherwise an 8-bit output.
template <typename X, typename RT, int K, bool kDrop>
__global__ void __launch_bounds__(kRowThreads, 1) fused_fwd_kernel(const FusedFwdParams p, const RowPlan pl) {
  constexpr bool kRes = Present<RT>::value;
  constexpr bool kQuant = !kDrop;
  constexpr int kStreams = kRes ? 2 : 1;
  RowCtx c = row_begin(pl, p.N);
  pdl_launch_dependents();
  pdl_wait();
  const void* src[kStreams];
  int bytes[kStreams];
  src[0] = p.x;
  bytes[0] = Vec8<X>::kBytes / 8;
  if constexpr (kRes) {
    src[1] = p.res;
    bytes[1] = Vec8<RT>::kBytes / 8;
  }
  const uint64_t policy = l2_policy_evict_first();
  if (c.gl == 0)
    for (int u = 0; u < pl.S && u < c.units; ++u) issue_unit(pl, c, u, u, p.rows, p.N, src, bytes, policy);
  load_affine(pl, c, p.w, p.w_dt, p.b, p.b_dt);
  const uint64_t offset = kDrop ? drop_offset(p.drop) : 0ull;
  const float inv_n = 1.f / static_cast<float>(p.N);
  const bool i8 = p.out_dt == RMSNORM_B200_I8;
  const float inv_q = i8 ? kInvI8 : kInvE4M3;
  const bool row_scale = kQuant && p.group == 0;
  const int scale_shift = kQuant && p.group ? 31 - __clz(p.group) : 0;

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
      uint32_t most = 0;
#pragma unroll
      for (int j = 0; j < K; ++j) {
        const int first_step = j & ~(pl.KC - 1);  // of this unit
        if (r == 0 && j == first_step) mbar_wait(&c.full[slot], phase, kSiteFwdFull);
        const int col = (j * pl.G + c.gl) * 8;
        if (col < c.ncols) {
          const unsigned char* base = c.ring + static_cast<size_t>(slot) * pl.unit_bytes;
          const int at = r * static_cast<int>(p.N) + col - first_step * pl.G * 8;
          Vec8<X>::load(base + at * (Vec8<X>::kBytes / 8), h[j]);
          float res[8];
          if constexpr (kRes) Vec8<RT>::load(base + pl.off[1] + at * (Vec8<RT>::kBytes / 8), res);
          if constexpr (kDrop) {
            const uint32_t keep = keep8(p.drop, c.slice0 + col, row, offset);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float base_v = kRes ? res[i] : 0.f;
              h[j][i] = keep >> i & 1u ? fmaf(h[j][i], p.drop.scale, base_v) : base_v;
            }
          } else if constexpr (kRes) {
#pragma unroll
            for (int i = 0; i < 8; ++i) h[j][i] += res[i];
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) ss = fmaf(h[j][i], h[j][i], ss);
          if (p.ro) store8_rt(p.ro, p.ro_dt, e0 + col, h[j]);
          if (row_scale && !pl.bias) {
            // max |y| = rstd * max |h w|: found along with the sum, one exchange for both
            float w[8];
            lds8(c.w + col, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) most = max(most, magnitude(h[j][i] * w[i]));
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) h[j][i] = 0.f;
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
      if (row_scale && !pl.bias)
        row_total<true, true>(pl, c, ss, most, kSiteFwdCluster);
      else
        row_total<true, false>(pl, c, ss, most, kSiteFwdCluster);
      const float rs = rsqrtf(ss * inv_n + p.eps);
      if (p.rstd && c.gl == 0 && c.rank == 0) st1(&p.rstd[row], rs);
      float inv = 1.f;     // of the row's scale: kept apart from rs, their product may overflow
      if (row_scale) {
        float largest;
        if (!pl.bias) {
          largest = __uint_as_float(most) * rs;
        } else {
#pragma unroll
          for (int j = 0; j < K; ++j) {
            const int col = (j * pl.G + c.gl) * 8;
            if (col < c.ncols) {
              float w[8], b[8];
              lds8(c.w + col, w);
              lds8(c.b + col, b);
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                h[j][i] = fmaf(h[j][i] * rs, w[i], b[i]);
                most = max(most, magnitude(h[j][i]));
              }
            }
          }
          float unused = 0.f;
          row_total<false, true>(pl, c, unused, most, kSiteFwdCluster);
          largest = __uint_as_float(most);
        }
        const float s = scale_of(largest, inv_q);
        if (c.gl == 0 && c.rank == 0) st1(&p.scales[row * p.scale_row], s);
        inv = 1.f / s;
      }
#pragma unroll
      for (int j = 0; j < K; ++j) {
        const int col = (j * pl.G + c.gl) * 8;
        const bool in = col < c.ncols;
        if (!__any_sync(0xffffffffu, in)) continue;
        float y[8];
        if (row_scale && pl.bias) {
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = h[j][i] * inv;
        } else {
          float w[8];
          if (in) {
            lds8(c.w + col, w);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = 0.f;
          }
          if (row_scale) {
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = (h[j][i] * w[i]) * rs * inv;
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = (h[j][i] * rs) * w[i];
            if (pl.bias && in) {
              float b[8];
              lds8(c.b + col, b);
#pragma unroll
              for (int i = 0; i < 8; ++i) y[i] = fmaf(h[j][i] * rs, w[i], b[i]);
            }
          }
        }
        if constexpr (kQuant) {
          if (!row_scale) {  // a scale's columns lie in 4, 8, 16 or 32 neighbouring lanes
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max(m, magnitude(y[i]));
            for (int o = p.group >> 4; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            const float s = scale_of(__uint_as_float(m), inv_q);
            const float inv_g = 1.f / s;
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] *= inv_g;
            const int64_t gcol = c.slice0 + col;
            if (in && (gcol & (p.group - 1)) == 0)
              st1(&p.scales[row * p.scale_row + (gcol >> scale_shift) * p.scale_group], s);
          }
          if (in) {
            uint2 q;
            if (i8) {
              q.x = to_i8(y[0]) | to_i8(y[1]) << 8 | to_i8(y[2]) << 16 | to_i8(y[3]) << 24;
              q.y = to_i8(y[4]) | to_i8(y[5]) << 8 | to_i8(y[6]) << 16 | to_i8(y[7]) << 24;
            } else {
              q.x = to_e4m3x2(y[0], y[1]) | to_e4m3x2(y[2], y[3]) << 16;
              q.y = to_e4m3x2(y[4], y[5]) | to_e4m3x2(y[6], y[7]) << 16;
            }
            uint2* dst = reinterpret_cast<uint2*>(static_cast<unsigned char*>(p.out) + e0 + col);
            if (RMSB_DBG_OK(dst, 8, kDbgVecStore)) __stcs(dst, q);
          }
        } else if (in) {
          store8_rt(p.out, p.out_dt, e0 + col, y);
        }
      }
    }
  }
  row_end(pl, c);
}

}  // namespace rmsb200
