// fused_fwd_kernels.cuh -- the streaming forward of the fused row operators.
#pragma once

#include "fused_generic.cuh"
#include "row_ring.cuh"

namespace rmsb200 {

// Vector steps a thread at most, and threads of a CTA. Four steps in 512 threads (128 registers
// each) beat two in 1024 for many rows: 8192 x 4096 bf16 + residual with 8-bit groups 43.8
// against 50.0 us, dropout 32768 x 4096 234 against 269 us. Few rows, a CTA each, take single
// steps in up to 1024 threads: 64 x 8192 5.7 against 6.7 us.
constexpr int kFwdSteps = 4;
constexpr int kFwdThreads = 512;
constexpr int kFwdFewThreads = 1024;

// What a row ends as.
struct Dropped {  // dropout; a floating output of x's type
  static constexpr bool kQuant = false, kRowScale = false;
};
template <typename Q, bool kRow>
struct Scaled {  // 8-bit values Q; one scale per row, or one per group of columns
  static constexpr bool kQuant = true, kRowScale = kRow;
  using Type = Q;
};

//   h = x + residual, or keep x / (1 - p) + residual;  y = h rsqrt(mean(h^2) + eps) w + b
//   8 bits: scale = max(largest |y| of the row or group / Q, 2^-126), q = round(y / scale)
// X, RT, ROT: types of x, of the residual and of residual_out (NoT: absent).
// A row is read once and stays in registers from its sum of squares to its output, so HBM sees
// 4 (8-bit output, no residual) to 12 bytes an element and nothing else. Measured with copies at
// 6.5 TB/s: 8 bits, one scale a row, bf16 + fp32 residual 32768 x 16384 725 to 795 us (738 us of
// bytes; the slower runs are under the power cap); scales of 128 columns, bf16 8192 x 4096 43 us
// (36 us of bytes, the rest the kernel's start and end); dropout, bf16 in, fp32 residual out,
// 32768 x 4096 216 us (205). Dropout between bf16 tensors is bound by the generator instead: 80
// instructions for 8 columns, 227 us for 164 us of bytes (72315 x 1856).
template <typename X, typename RT, typename ROT, typename End, int K>
__global__ void __launch_bounds__(K == 1 ? kFwdFewThreads : kFwdThreads, 1)
    fused_fwd_kernel(const FusedFwdParams p, const RowPlan pl) {
  constexpr bool kRes = Present<RT>::value, kRo = Present<ROT>::value;
  constexpr bool kQuant = End::kQuant, kRowScale = End::kRowScale;
  constexpr int kStreams = kRes ? 2 : 1;
  constexpr int kX = Vec8<X>::kBytes / 8;
  RowCtx c = row_begin(pl, p.N);
  pdl_launch_dependents();
  pdl_wait();
  const void* src[kStreams];
  int bytes[kStreams];
  src[0] = p.x;
  bytes[0] = kX;
  if constexpr (kRes) {
    src[1] = p.res;
    bytes[1] = Vec8<RT>::kBytes / 8;
  }
  const uint64_t policy = l2_policy_evict_first();
  if (c.gl == 0)
    for (int u = 0; u < pl.S && u < c.units; ++u) issue_unit(pl, c, u, u, p.rows, p.N, src, bytes, policy);
  load_affine(pl, c, p.w, p.w_dt, p.b, p.b_dt);
  const uint64_t offset = kQuant ? 0ull : drop_offset(p.drop);
  const float inv_n = 1.f / static_cast<float>(p.N);

  int slot = 0;
  uint32_t phase = 0;
  int64_t unit = 0;
  for (int64_t tile = c.first; tile < pl.tiles; tile += c.step) {
    const int64_t row0 = tile * pl.R;
    const int nrows = static_cast<int>(min(static_cast<int64_t>(pl.R), p.rows - row0));
    for (int r = 0; r < nrows; ++r) {
      const int64_t row = row0 + r;
      const int64_t e0 = row * p.N + c.slice0;
      float2 h[K][4];  // h; with a row's scale and no bias, h w
      float2 ss = make_float2(0.f, 0.f);
      float most = 0.f;
#pragma unroll
      for (int j = 0; j < K; ++j) {
        const int first_step = j & ~(pl.KC - 1);  // of this unit
        if (r == 0 && j == first_step) mbar_wait_warp(&c.full[slot], phase, kSiteFwdFull);
        const int col = (j * pl.G + c.gl) * 8;
        if (col < c.ncols) {
          const unsigned char* base = c.ring + static_cast<size_t>(slot) * pl.unit_bytes;
          const int at = r * static_cast<int>(p.N) + col - first_step * pl.G * 8;
          Pair8<X>::load(base + at * kX, h[j]);
          float2 res[4];
          if constexpr (kRes) Pair8<RT>::load(base + pl.off[1] + at * (Vec8<RT>::kBytes / 8), res);
          if constexpr (!kQuant) {
            if constexpr (!kRes)
              for (float2& v : res) v = make_float2(0.f, 0.f);
            float2 kept[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) kept[i] = fma2(h[j][i], splat2(p.drop.scale), res[i]);
            uint32_t words[2][4];
            draw8(p.drop, c.slice0 + col, row, offset, words);
            select8(p.drop, words, kept, res, h[j]);
          } else if constexpr (kRes) {
#pragma unroll
            for (int i = 0; i < 4; ++i) h[j][i] = add2(h[j][i], res[i]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) ss = fma2(h[j][i], h[j][i], ss);
          if constexpr (kRo)
            Pair8<ROT>::store(static_cast<unsigned char*>(p.ro) + (e0 + col) * (Vec8<ROT>::kBytes / 8), h[j]);
          if (kRowScale && !pl.bias) {
            // max |y| = rstd * max |h w|: found along with the sum, one exchange for both
            float2 w[4];
            affine8(pl, c.w, col, w);
#pragma unroll
            for (int i = 0; i < 4; ++i) h[j][i] = mul2(h[j][i], w[i]);
            most = largest8(most, h[j]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) h[j][i] = make_float2(0.f, 0.f);
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
      float sum = ss.x + ss.y;
      uint32_t bits = magnitude(most);
      if (kRowScale && !pl.bias)
        row_total<true, true>(pl, c, sum, bits, kSiteFwdCluster);
      else
        row_total<true, false>(pl, c, sum, bits, kSiteFwdCluster);
      const float rs = rsqrtf(sum * inv_n + p.eps);
      if (p.rstd && c.gl == 0 && c.rank == 0) st1(&p.rstd[row], rs);
      // y in the place of h
#pragma unroll
      for (int j = 0; j < K; ++j) {
        const int col = (j * pl.G + c.gl) * 8;
        if (col >= c.ncols) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i) h[j][i] = mul2(h[j][i], splat2(rs));
        if (kRowScale && !pl.bias) continue;
        float2 w[4];
        affine8(pl, c.w, col, w);
        if (pl.bias) {
          float2 b[4];
          affine8(pl, c.b, col, b);
#pragma unroll
          for (int i = 0; i < 4; ++i) h[j][i] = fma2(h[j][i], w[i], b[i]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) h[j][i] = mul2(h[j][i], w[i]);
        }
        if constexpr (!kQuant)
          Pair8<X>::store(static_cast<unsigned char*>(p.out) + (e0 + col) * kX, h[j]);
      }
      if constexpr (kQuant) {
        using Q = typename End::Type;
        float inv[K];
        if constexpr (kRowScale) {
          float largest = __uint_as_float(bits) * rs;
          if (pl.bias) {
            most = 0.f;
#pragma unroll
            for (int j = 0; j < K; ++j) most = largest8(most, h[j]);
            bits = magnitude(most);
            float unused = 0.f;
            row_total<false, true>(pl, c, unused, bits, kSiteFwdCluster);
            largest = __uint_as_float(bits);
          }
          const float s = scale_of(largest, Q::kInvQ);
          if (c.gl == 0 && c.rank == 0) st1(&p.scales[row * p.scale_row], s);
#pragma unroll
          for (int j = 0; j < K; ++j) inv[j] = inverse(s);
        } else {  // a scale's columns lie in 4, 8, 16 or 32 neighbouring lanes
          float m[K];
#pragma unroll
          for (int j = 0; j < K; ++j) m[j] = largest8(0.f, h[j]);
          for (int o = p.group >> 4; o > 0; o >>= 1) {
#pragma unroll
            for (int j = 0; j < K; ++j) m[j] = max3_abs(m[j], __shfl_xor_sync(0xffffffffu, m[j], o), 0.f);
          }
#pragma unroll
          for (int j = 0; j < K; ++j) {
            const int col = (j * pl.G + c.gl) * 8;
            const float s = scale_of(m[j], Q::kInvQ);
            inv[j] = inverse(s);
            if (col < c.ncols && (col & (p.group - 1)) == 0)  // slices begin at whole groups
              st1(&p.scales[row * p.scale_row + ((c.slice0 + col) >> p.group_shift) * p.scale_group], s);
          }
        }
#pragma unroll
        for (int j = 0; j < K; ++j) {
          const int col = (j * pl.G + c.gl) * 8;
          if (col >= c.ncols) continue;
#pragma unroll
          for (int i = 0; i < 4; ++i) h[j][i] = mul2(h[j][i], splat2(inv[j]));
          uint2* dst = reinterpret_cast<uint2*>(static_cast<unsigned char*>(p.out) + e0 + col);
          if (RMSB_DBG_OK(dst, 8, kDbgVecStore))
            __stcs(dst, make_uint2(Q::pack4(h[j][0], h[j][1]), Q::pack4(h[j][2], h[j][3])));
        }
      }
    }
  }
  row_end(pl, c);
}

}  // namespace rmsb200
