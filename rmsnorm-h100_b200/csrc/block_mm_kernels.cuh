// block_mm_kernels.cuh -- products of e4m3 matrices whose values have an fp32 scale per group of
// 128 columns (block_mm.cu chooses among them).
//
//   out[m][n] = sum_g a_scale[m][g] b_scale[n][g] sum_{k in g} a[m][k] b[n][k]  (+ bias[n])
//
// The tensor cores sum one group of 128 columns at a time into tensor memory; a scale holds for a
// group, so the sum over the groups is made outside of them, in registers and in fp32, while the
// next group is on its way: a multiply-add for every element and group, and a multiplication more
// where b has a scale a row.
#pragma once

#include "block_scale.cuh"
#include "tensor_core.cuh"

namespace rmsb200 {

constexpr int kSiteMmFull = 13, kSiteMmEmpty = 14, kSiteMmSum = 15, kSiteMmSumEmpty = 16;  // waits that gave up

struct BlockMmParams {
  int64_t m;
  int32_t n, groups;
  const float* sa;
  int64_t sa_row, sa_group;
  const float* sb;
  int64_t sb_row, sb_group;
  const void* bias;
  void* out;
  int32_t bias_dt, out_dt;
  bool b_rows;      // b's scales are per row
  bool vec_out;     // out's rows begin at multiples of 32 bytes
  bool vec_bias;    // bias begins at one of 16
};

__device__ __forceinline__ const float* sb_of(const BlockMmParams& p, int64_t n) {
  return p.sb + (p.b_rows ? n : n / kBlock) * p.sb_row;
}

// ---------------------------------------------------------------------------------------
// Many rows: 256 x 256 of the result a pair of CTAs, whose tensor cores work on one product: each
// CTA holds 128 rows of a and of b and half of the result, so that what both need of b crosses
// from L2 once. Tensor memory holds two groups' sums (all of it), so a group's have to be taken out
// within the time of the next one's products.
// Measured (bf16 results, in a burst): 8192 x 16384 x 4096 495 to 510 us, 2160 to 2220 TFLOP/s; with
// a scale a row of b, whose exchange has the summing warps meet once a group, 8192 x 4096 x 8192 345
// to 395 us (blocks: 243 us). The products alone run at 3950 TFLOP/s, with
// their copies at 2860 (the card's power limit), with the sums' hand-over as well at 2460, with
// tensor memory read at 2270: the scaling shares its time with none of these completely.
// What was tried: accumulators of 128 columns, four of them, 575 us and more; 16 summing warps of
// 64 columns 519 us; 32 columns at a time out of tensor memory 514 us; single CTAs 570 us.
// ---------------------------------------------------------------------------------------
constexpr int kWideRows = 256, kWideN = 256;  // rows and columns of a pair's tile
constexpr int kWideThreads = 384;  // warps 0 - 7 sum, 8 copies, 9 multiplies
constexpr int kWideHalf = kWideN / 2;
constexpr int kTileBytes = kBlock * kTileK;  // 128 rows of an operand

constexpr int kWideStages = 6;
constexpr int kWideStageBytes = 2 * kTileBytes;  // a CTA's rows of a and of b

constexpr int kStagingBytes = 32 * 17 * 4;  // store_turned's: 32 rows of 16 columns, a word between them

struct WideBars {
  uint64_t full[kWideStages], empty[kWideStages], sum[2], sum_empty[2], done;
  uint32_t tmem;
};

struct WidePlan {
  int32_t tiles_m, tiles_n, band;  // tiles go down `band` rows of tiles before the next column
};

__device__ __forceinline__ void wide_tile(const WidePlan& pl, int64_t i, int* tm, int* tn) {
  const int64_t per = static_cast<int64_t>(pl.band) * pl.tiles_n;
  const int b = static_cast<int>(i / per);
  const int64_t at = i - b * per;
  const int high = min(pl.band, pl.tiles_m - b * pl.band);
  *tn = static_cast<int>(at / high);
  *tm = b * pl.band + static_cast<int>(at - static_cast<int64_t>(*tn) * high);
}

// A whole 32-byte sector: a lane's neighbours write other rows.
__device__ __forceinline__ void store32(void* p, const uint32_t (&w)[8]) {
  if (!RMSB_DBG_OK(p, 32, kDbgVecStore)) return;
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// A warp's 32 rows of 16 columns, a row a lane, where rows begin anywhere: turned through shared
// memory, so that the warp stores a row's neighbours side by side (1000 x 4100 with K = 1008: 50 us
// when every lane stored its own row's values one by one, 14 us so).
__device__ __forceinline__ void store_turned(float* mine, const float2 (&v)[8], const BlockMmParams& p, int64_t row0,
                                             int64_t col0, int left) {
  const int rows = static_cast<int>(max(int64_t{0}, min(int64_t{32}, p.m - row0)));
  const int lane = threadIdx.x & 31;
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 16; ++i) mine[lane * 17 + i] = i & 1 ? v[i / 2].y : v[i / 2].x;
  __syncwarp();
  const int col = lane & 15;
  if (col >= left) return;
  const float bias = p.bias ? load1_rt(p.bias, p.bias_dt, col0 + col) : 0.f;
  for (int r = lane >> 4; r < rows; r += 2)
    store1_rt(p.out, p.out_dt, (row0 + r) * p.n + col0 + col, mine[r * 17 + col] + bias);
}

// Adds bias to 16 columns from col on, a multiple of 16.
__device__ __forceinline__ void add_bias16(const BlockMmParams& p, int64_t col, float2* v) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float2 b[4];
    if (p.vec_bias) {
      load8p_rt(p.bias, p.bias_dt, col + 8 * k, b);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        b[i] = make_float2(load1_rt(p.bias, p.bias_dt, col + 8 * k + 2 * i), load1_rt(p.bias, p.bias_dt, col + 8 * k + 2 * i + 1));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[4 * k + i] = add2(v[4 * k + i], b[i]);
  }
}

// What a chunk's sums are multiplied by: scale, or (column scales) * scale. The two scales first, as
// wherever they are multiplied, so that only their product has to be a number of fp32.
template <bool kRowScales>
__device__ __forceinline__ void chunk_scales(float2 (&to)[8], float s, const float* col) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    if constexpr (kRowScales) {
      const float4 c = *reinterpret_cast<const float4*>(col + 2 * i);
      to[i] = mul2(make_float2(c.x, c.y), splat2(s));
      to[i + 1] = mul2(make_float2(c.z, c.w), splat2(s));
    } else {
      to[i] = to[i + 1] = splat2(s);
    }
  }
}

template <bool kRowScales>
__global__ void __launch_bounds__(kWideThreads, 1)
    block_mm_wide_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                         const BlockMmParams p, const WidePlan pl) {
  unsigned char* smem = rmsb_dyn_smem + ((1024u - (smem_u32(rmsb_dyn_smem) & 1023u)) & 1023u);
  WideBars* bars = reinterpret_cast<WideBars*>(smem + kWideStages * kWideStageBytes);
  float* col_scales = reinterpret_cast<float*>(bars + 1);  // [2][kWideN]
  unsigned char* staging = reinterpret_cast<unsigned char*>(col_scales + 2 * kWideN);  // kStagingBytes a warp
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int64_t unit = blockIdx.x >> 1, units = gridDim.x >> 1;
  const int64_t tiles = static_cast<int64_t>(pl.tiles_m) * pl.tiles_n;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kWideStages; ++i) {
      mbar_init(&bars->full[i], 1);
      mbar_init(&bars->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->sum[i], 1);
      mbar_init(&bars->sum_empty[i], 16);
    }
    mbar_init(&bars->done, 1);
    fence_mbar_init();
  }
  if (warp == 9) tmem_alloc_pair(&bars->tmem, 2 * kWideN);
  if (threadIdx.x == 256) {
    prefetch_map(&map_a);
    prefetch_map(&map_b);
  }
  tmem_fence_before_sync();
  __syncthreads();
  cluster_sync_all();
  tmem_fence_after_sync();
  const uint32_t tmem = bars->tmem;
  pdl_launch_dependents();  // they may take tensor memory and wait: this grid has all of its own by now
  pdl_wait();

  if (warp >= 8) {
    regs_down<40>();
    if (warp == 8) {  // copies
      int s = 0;
      uint32_t pass = 0;
      bool ok = true;
      for (int64_t t = unit; ok && t < tiles; t += units) {
        int tm, tn;
        wide_tile(pl, t, &tm, &tn);
        const int ya = tm * kWideRows + static_cast<int>(rank) * kBlock;
        const int yb = tn * kWideN + static_cast<int>(rank) * kBlock;
        for (int g = 0; g < p.groups; ++g) {
          ok = __all_sync(0xffffffffu, mbar_spin_warp(&bars->empty[s], pass ^ 1u, kSiteMmEmpty));
          if (!ok) break;
          if (elect_one()) {
            unsigned char* at = smem + s * kWideStageBytes;
            if (rank == 0) mbar_arrive_expect_tx(&bars->full[s], 2 * kWideStageBytes);
            tile_load<true>(at, &map_a, g * kTileK, ya, &bars->full[s]);
            tile_load<true>(at + kTileBytes, &map_b, g * kTileK, yb, &bars->full[s]);
          }
          __syncwarp();
          if (++s == kWideStages) {
            s = 0;
            pass ^= 1u;
          }
        }
      }
      // Nobody leaves while copies may land in its memory or arrivals at its barriers.
      if (lane == 0 && rank == 0 && abort_requested())
        for (int i = 0; i < kWideStages; ++i) mbar_wait(&bars->full[i], i < s ? pass : pass ^ 1u, kSiteDrain, false);
      for (int i = 0; i < kWideStages; ++i) mbar_spin_warp(&bars->empty[i], i < s ? pass : pass ^ 1u, kSiteMmEmpty);
    } else if (warp == 9 && rank == 0) {  // products
      constexpr uint32_t idesc = product_desc(kWideRows, kWideN);
      int s = 0;
      uint32_t pass = 0, u = 0;
      bool ok = true;
      for (int64_t t = unit; ok && t < tiles; t += units)
        for (int g = 0; g < p.groups; ++g, ++u) {
          const uint32_t d = u & 1u;
          ok = mbar_spin_warp(&bars->full[s], pass, kSiteMmFull);
          ok = mbar_spin_warp(&bars->sum_empty[d], ((u >> 1) & 1u) ^ 1u, kSiteMmSumEmpty) && ok;
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tmem_fence_after_sync();
          if (elect_one()) {
            const uint32_t at = smem_u32(smem + s * kWideStageBytes);
            const uint64_t a = operand_desc(at), b = operand_desc(at + kTileBytes);
#pragma unroll
            for (int k = 0; k < kTileK / 32; ++k) mma_e4m3<true>(tmem + d * kWideN, a + 2 * k, b + 2 * k, idesc, k > 0);
            mma_commit<true>(&bars->empty[s]);
            mma_commit<true>(&bars->sum[d]);
          }
          __syncwarp();
          if (++s == kWideStages) {
            s = 0;
            pass ^= 1u;
          }
        }
      if (__any_sync(0xffffffffu, abort_requested())) {  // the products issued so far end first
        if (elect_one()) mma_commit<true>(&bars->done);
        __syncwarp();
        if (lane == 0) mbar_wait(&bars->done, 0, kSiteDrain, false);
        __syncwarp();
      }
      for (int i = 0; i < 2; ++i, ++u) mbar_spin_warp(&bars->sum_empty[u & 1u], ((u >> 1) & 1u) ^ 1u, kSiteMmSumEmpty);
    }
  } else {  // sums: warp w has rows 32 (w % 4) .. + 31, the half w / 4 of the columns
    regs_up<232>();
    const int half = warp >> 2;
    const uint32_t from = tmem + (static_cast<uint32_t>(warp & 3) << 21) + half * kWideHalf;
    uint32_t u = 0;
    for (int64_t t = unit; t < tiles; t += units) {
      int tm, tn;
      wide_tile(pl, t, &tm, &tn);
      const int64_t row = static_cast<int64_t>(tm) * kWideRows + rank * kBlock + (warp & 3) * 32 + lane;
      const int64_t col0 = static_cast<int64_t>(tn) * kWideN + half * kWideHalf;
      const bool live = row < p.m;
      // scales kAhead groups ahead; b's per row: thread i of the 256 brings column i's, else every
      // thread its half's
      const int64_t own = kRowScales ? static_cast<int64_t>(tn) * kWideN + threadIdx.x : col0;
      const bool own_live = own < p.n;
      const float* sa = p.sa + row * p.sa_row;
      const float* sb = sb_of(p, own);
      auto next_a = [&](int g) {
        const float v = live && g < p.groups ? ld1(sa) : 0.f;
        sa += p.sa_group;
        return v;
      };
      auto next_b = [&](int g) {
        const float v = own_live && g < p.groups ? ld1(sb) : 0.f;
        sb += p.sb_group;
        return v;
      };
      constexpr int kAhead = 2;
      float a[kAhead], b[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        a[i] = next_a(i);
        b[i] = next_b(i);
      }
      float2 acc[kWideHalf / 2];
#pragma unroll
      for (int i = 0; i < kWideHalf / 2; ++i) acc[i] = make_float2(0.f, 0.f);
      for (int g = 0; g < p.groups; ++g, ++u) {
        const uint32_t d = u & 1u;
        float s = a[0];
        const float* cols = col_scales + d * kWideN;
        if constexpr (kRowScales) {
          col_scales[d * kWideN + threadIdx.x] = b[0];
          __syncwarp();
          named_barrier(1, 256);
          cols += half * kWideHalf;
        } else {
          s *= b[0];
        }
#pragma unroll
        for (int i = 0; i + 1 < kAhead; ++i) {
          a[i] = a[i + 1];
          b[i] = b[i + 1];
        }
        a[kAhead - 1] = next_a(g + kAhead);
        b[kAhead - 1] = next_b(g + kAhead);
        mbar_spin_warp(&bars->sum[d], (u >> 1) & 1u, kSiteMmSum);
        __syncwarp();
        tmem_fence_after_sync();
        const uint32_t at = from + d * kWideN;
        float2 v[2][8], scale[8];
        tmem_ld(at, v[0]);
        chunk_scales<kRowScales>(scale, s, cols);  // a chunk's while its sums are on their way
        tmem_landed(v[0]);
#pragma unroll
        for (int c = 0; c < kWideHalf / 16; ++c) {
          if (c + 1 < kWideHalf / 16) tmem_ld(at + (c + 1) * 16, v[(c + 1) & 1]);
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[8 * c + i] = fma2(v[c & 1][i], scale[i], acc[8 * c + i]);
          if (c + 1 < kWideHalf / 16) chunk_scales<kRowScales>(scale, s, cols + 16 * (c + 1));
          if (c + 1 < kWideHalf / 16) tmem_landed(v[(c + 1) & 1]);
          if (c + 2 == kWideHalf / 16) {
            tmem_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive_peer(&bars->sum_empty[d], 0);
          }
        }
      }
      const int64_t e = row * p.n + col0;
      const int left = static_cast<int>(min(static_cast<int64_t>(kWideHalf), p.n - col0));
      if (!p.vec_out || left < kWideHalf) {
        float* mine = reinterpret_cast<float*>(staging + warp * kStagingBytes);
#pragma unroll
        for (int c = 0; c < kWideHalf; c += 16) {
          float2 v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = acc[c / 2 + i];
          if (c < left) store_turned(mine, v, p, row - lane, col0 + c, left - c);
        }
        continue;
      }
      if (!live) continue;
      if (p.bias) {
#pragma unroll
        for (int c = 0; c < kWideHalf; c += 16) add_bias16(p, col0 + c, acc + c / 2);
      }
      if (p.out_dt == RMSNORM_B200_F32) {
        float* out = static_cast<float*>(p.out) + e;
#pragma unroll
        for (int i = 0; i < kWideHalf; i += 8) {
          uint32_t w[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) w[k] = __float_as_uint(k & 1 ? acc[(i + k) / 2].y : acc[(i + k) / 2].x);
          store32(out + i, w);
        }
      } else {
        uint16_t* out = static_cast<uint16_t*>(p.out) + e;
        const bool bf16 = p.out_dt == RMSNORM_B200_BF16;
#pragma unroll
        for (int i = 0; i < kWideHalf; i += 16) {
          uint32_t w[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) w[k] = bf16 ? pack_bf16x2_pair(acc[i / 2 + k]) : pack_f16x2_pair(acc[i / 2 + k]);
          store32(out + i, w);
        }
      }
    }
  }
  __syncwarp();
  tmem_fence_before_sync();
  __syncthreads();
  cluster_sync_all();
  tmem_fence_after_sync();
  if (warp == 9) tmem_dealloc_pair(tmem, 2 * kWideN);
}

// ---------------------------------------------------------------------------------------
// Many rows, scales that are powers of two, 16-bit results: the tensor cores apply the scales.
// Warps 10 to 13 turn a group's scales into exponents, one for every 32 values of k, which a copy
// in the products' order brings to tensor memory; the sum over all of k stays there, and the eight
// summing warps only bring results out. Tiles of 224 or 192 columns leave tensor memory for two of
// them, so that one comes out while the next is summed, and for the exponents; one of 256 comes out
// before the next begins, for pairs that have a single tile or two. Each addition of 32 products
// rounds towards zero: where all values are positive, sums are low by 9.1e-6, 3.9e-5 and 3.3e-4 of
// themselves at 4096, 16384 and 131072 columns (scaled in registers: 1e-7 to 5e-7).
// Measured in a burst: 8192 x 16384 x 4096 409 us (2690 TFLOP/s, at the card's power limit), scaled
// in registers 495 to 510 us.
// ---------------------------------------------------------------------------------------
constexpr int kScaledThreads = 448;
constexpr int kScaledStages = 6;
constexpr int kExpBytes = 3 * 512;  // exponents of a stage: of 128 rows of a, 256 of b
constexpr int kExpAhead = 8;        // groups whose scales are on their way

template <int N>
struct ScaledTile {
  static constexpr int kSums = N > 224 ? 1 : 2;
  static constexpr int kStageBytes = kTileBytes + N / 2 * kTileK;  // a CTA's rows of a and of b
  static constexpr int kExpColumns = kSums * N;                    // in tensor memory, 16 columns for each of four groups
};

struct ScaledBars {
  uint64_t full[kScaledStages], empty[kScaledStages], sum[2], sum_empty[2], done;
  uint32_t tmem;
};

template <int N>
__global__ void __launch_bounds__(kScaledThreads, 1)
    block_mm_scaled_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                           const BlockMmParams p, const WidePlan pl) {
  using S = ScaledTile<N>;
  unsigned char* smem = rmsb_dyn_smem + ((1024u - (smem_u32(rmsb_dyn_smem) & 1023u)) & 1023u);
  unsigned char* exponents = smem + kScaledStages * S::kStageBytes;
  ScaledBars* bars = reinterpret_cast<ScaledBars*>(exponents + kScaledStages * kExpBytes);
  unsigned char* staging = reinterpret_cast<unsigned char*>(bars + 1);  // kStagingBytes a warp
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int64_t unit = blockIdx.x >> 1, units = gridDim.x >> 1;
  const int64_t tiles = static_cast<int64_t>(pl.tiles_m) * pl.tiles_n;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kScaledStages; ++i) {
      mbar_init(&bars->full[i], 9);  // the copies, and four warps' exponents in each CTA
      mbar_init(&bars->empty[i], 1);
    }
    for (int i = 0; i < S::kSums; ++i) {
      mbar_init(&bars->sum[i], 1);
      mbar_init(&bars->sum_empty[i], 16);
    }
    mbar_init(&bars->done, 1);
    fence_mbar_init();
  }
  if (warp == 9) tmem_alloc_pair(&bars->tmem, 512);
  if (threadIdx.x == 256) {
    prefetch_map(&map_a);
    prefetch_map(&map_b);
  }
  tmem_fence_before_sync();
  __syncthreads();
  cluster_sync_all();
  tmem_fence_after_sync();
  const uint32_t tmem = bars->tmem;
  pdl_launch_dependents();  // they may take tensor memory and wait: this grid has all of its own by now
  pdl_wait();

  if (warp == 8) {  // copies
    int s = 0;
    uint32_t pass = 0;
    bool ok = true;
    for (int64_t t = unit; ok && t < tiles; t += units) {
      int tm, tn;
      wide_tile(pl, t, &tm, &tn);
      const int ya = tm * kWideRows + static_cast<int>(rank) * kBlock;
      const int yb = tn * N + static_cast<int>(rank) * (N / 2);
      for (int g = 0; g < p.groups; ++g) {
        ok = __all_sync(0xffffffffu, mbar_spin_warp(&bars->empty[s], pass ^ 1u, kSiteMmEmpty));
        if (!ok) break;
        if (elect_one()) {
          unsigned char* at = smem + s * S::kStageBytes;
          if (rank == 0) mbar_arrive_expect_tx(&bars->full[s], 2 * S::kStageBytes);
          tile_load<true>(at, &map_a, g * kTileK, ya, &bars->full[s]);
          tile_load<true>(at + kTileBytes, &map_b, g * kTileK, yb, &bars->full[s]);
        }
        __syncwarp();
        if (++s == kScaledStages) {
          s = 0;
          pass ^= 1u;
        }
      }
    }
    // Nobody leaves while copies may land in its memory or arrivals at its barriers.
    if (lane == 0 && rank == 0 && abort_requested())
      for (int i = 0; i < kScaledStages; ++i) mbar_wait(&bars->full[i], i < s ? pass : pass ^ 1u, kSiteDrain, false);
    for (int i = 0; i < kScaledStages; ++i) mbar_spin_warp(&bars->empty[i], i < s ? pass : pass ^ 1u, kSiteMmEmpty);
  } else if (warp == 9 && rank == 0) {  // products
    constexpr uint32_t idesc = scaled_product_desc(kWideRows, N);
    int s = 0;
    uint32_t pass = 0, u = 0, n = 0;  // rounds of the stages, tiles, groups
    bool ok = true;
    for (int64_t t = unit; ok && t < tiles; t += units, ++u) {
      const uint32_t d = u % S::kSums;
      ok = __all_sync(0xffffffffu, mbar_spin_warp(&bars->sum_empty[d], ((u / S::kSums) & 1u) ^ 1u, kSiteMmSumEmpty));
      for (int g = 0; ok && g < p.groups; ++g, ++n) {
        ok = __all_sync(0xffffffffu, mbar_spin_warp(&bars->full[s], pass, kSiteMmFull));
        if (!ok) break;
        tmem_fence_after_sync();
        if (elect_one()) {
          const uint32_t at = smem_u32(smem + s * S::kStageBytes), exps = smem_u32(exponents + s * kExpBytes);
          const uint32_t sa = tmem + S::kExpColumns + (n & 3u) * 16, sb = sa + 4;
          scales_to_tmem(sa, exps);
          scales_to_tmem(sb, exps + 512);
          scales_to_tmem(sb + 4, exps + 1024);
          const uint64_t a = operand_desc(at), b = operand_desc(at + kTileBytes);
#pragma unroll
          for (int k = 0; k < kTileK / 32; ++k)
            mma_e4m3_scaled(tmem + d * N, a + 2 * k, b + 2 * k, idesc, sa, sb, g > 0 || k > 0);
          mma_commit<true>(&bars->empty[s]);
          if (g == p.groups - 1) mma_commit<true>(&bars->sum[d]);
        }
        __syncwarp();
        if (++s == kScaledStages) {
          s = 0;
          pass ^= 1u;
        }
      }
    }
    if (__any_sync(0xffffffffu, abort_requested())) {  // the products issued so far end first
      if (elect_one()) mma_commit<true>(&bars->done);
      __syncwarp();
      if (lane == 0) mbar_wait(&bars->done, 0, kSiteDrain, false);
      __syncwarp();
    }
    for (int i = 0; i < S::kSums; ++i, ++u)
      mbar_spin_warp(&bars->sum_empty[u % S::kSums], ((u / S::kSums) & 1u) ^ 1u, kSiteMmSumEmpty);
  } else if (warp >= 10) {  // exponents: thread i has row i of a, rows i and i + 128 of b
    const int i = threadIdx.x - 320;
    int s = 0;
    uint32_t pass = 0;
    for (int64_t t = unit; t < tiles; t += units) {
      int tm, tn;
      wide_tile(pl, t, &tm, &tn);
      const int64_t rows[3] = {static_cast<int64_t>(tm) * kWideRows + rank * kBlock + i, static_cast<int64_t>(tn) * N + i,
                               static_cast<int64_t>(tn) * N + i + 128};
      const bool live[3] = {rows[0] < p.m, rows[1] < p.n, rows[2] < p.n && i + 128 < N};
      const float* src[3] = {p.sa + rows[0] * p.sa_row, sb_of(p, rows[1]), sb_of(p, rows[2])};
      int ahead = 0;
      auto fetch = [&](uint32_t (&e)[3]) {
#pragma unroll
        for (int j = 0; j < 3; ++j) {
          e[j] = live[j] && ahead < p.groups ? __float_as_uint(ld1(src[j])) : 0x3f800000u;
          src[j] += j < 1 ? p.sa_group : p.sb_group;
        }
        ++ahead;
      };
      uint32_t e[kExpAhead][3];
#pragma unroll
      for (int k = 0; k < kExpAhead; ++k) fetch(e[k]);
      for (int g = 0; g < p.groups; ++g) {
        uint32_t word[3];
#pragma unroll
        for (int j = 0; j < 3; ++j) {
          word[j] = (e[0][j] >> 23 & 255u) * 0x01010101u;
#pragma unroll
          for (int k = 1; k < kExpAhead; ++k) e[k - 1][j] = e[k][j];
        }
        fetch(e[kExpAhead - 1]);
        mbar_spin_warp(&bars->empty[s], pass ^ 1u, kSiteMmEmpty);
        uint32_t* to = reinterpret_cast<uint32_t*>(exponents + s * kExpBytes) + (i & 31) * 4 + (i >> 5);
#pragma unroll
        for (int j = 0; j < 3; ++j) to[128 * j] = word[j];
        // The bytes are in place for this SM's tensor core before the arrival leaves; the pair's
        // first CTA makes it read them. (Release at the cluster's scope would wait for the loads in
        // flight: 1058 instead of 460 us at 8192 x 16384 x 4096.)
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive_peer(&bars->full[s], 0);
        if (++s == kScaledStages) {
          s = 0;
          pass ^= 1u;
        }
      }
    }
  } else if (warp < 8) {  // results: warp w has rows 32 (w % 4) .. + 31, the half w / 4 of the columns
    constexpr int kHalf = N / 2;
    const int half = warp >> 2;
    const uint32_t from = tmem + (static_cast<uint32_t>(warp & 3) << 21) + half * kHalf;
    uint32_t u = 0;
    for (int64_t t = unit; t < tiles; t += units, ++u) {
      int tm, tn;
      wide_tile(pl, t, &tm, &tn);
      const uint32_t d = u % S::kSums;
      const int64_t row = static_cast<int64_t>(tm) * kWideRows + rank * kBlock + (warp & 3) * 32 + lane;
      const int64_t col0 = static_cast<int64_t>(tn) * N + half * kHalf;
      const int left = static_cast<int>(max(int64_t{0}, min(static_cast<int64_t>(kHalf), p.n - col0)));
      const bool whole = p.vec_out && left == kHalf, bf16 = p.out_dt == RMSNORM_B200_BF16;
      mbar_spin_warp(&bars->sum[d], (u / S::kSums) & 1u, kSiteMmSum);
      __syncwarp();
      tmem_fence_after_sync();
#pragma unroll
      for (int c = 0; c < kHalf; c += 16) {
        float2 v[8];
        __syncwarp();  // of the chunk before, lanes stored or did not
        tmem_ld(from + d * N + c, v);
        tmem_landed(v);
        if (c + 16 == kHalf) {
          tmem_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive_peer(&bars->sum_empty[d], 0);
        }
        if (c >= left) continue;
        if (whole) {
          if (p.bias) add_bias16(p, col0 + c, v);
          if (row < p.m) {
            uint32_t w[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) w[k] = bf16 ? pack_bf16x2_pair(v[k]) : pack_f16x2_pair(v[k]);
            store32(static_cast<uint16_t*>(p.out) + row * p.n + col0 + c, w);
          }
        } else {
          store_turned(reinterpret_cast<float*>(staging + warp * kStagingBytes), v, p, row - lane, col0 + c, left - c);
        }
      }
    }
  }
  __syncwarp();
  tmem_fence_before_sync();
  __syncthreads();
  cluster_sync_all();
  tmem_fence_after_sync();
  if (warp == 9) tmem_dealloc_pair(tmem, 512);
}

// ---------------------------------------------------------------------------------------
// Few rows: the rows of b take the tensor cores' 128 rows and the T rows of a their columns, so
// that b streams through once. The groups of k are split over the CTAs of a cluster, each of
// which then adds up some rows of the result.
// Measured: 1 x 16384 x 16384 46 us (5.8 TB/s), 8 x 16384 x 4096 14.7 us (4.6), 64 x 8192 x 8192
// 17.3 us (4.0), 1 x 4096 x 4096 5.9 to 7 us: start, the way of the first copies and the joining of
// the parts take 5 to 6 us of each.
// ---------------------------------------------------------------------------------------
constexpr int kFewThreads = 192;  // warps 0 - 3 sum, 4 copies, 5 multiplies
constexpr int kFewMaxStages = 16, kFewMaxSplits = 8, kFewChunk = 16;

template <int T>
struct Few {
  static constexpr int kSums = T >= 128 ? 2 : 4;
  static constexpr int kTmem = kSums * T;  // columns: a power of two, at least 32
  static constexpr int kStageBytes = kTileBytes + T * kTileK;
};

struct FewBars {
  uint64_t full[kFewMaxStages], empty[kFewMaxStages], sum[4], sum_empty[4], done;
  uint32_t tmem;
};

struct FewPlan {
  int32_t tiles_n, splits, stages;
  int32_t ring_bytes;  // of the stages, and room for the sums that take their place
};

template <int T>
__global__ void __launch_bounds__(kFewThreads, T >= 128 ? 1 : 2)
    block_mm_few_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                        const BlockMmParams p, const FewPlan pl) {
  using F = Few<T>;
  constexpr int kChunk = T < 32 ? 16 : 32;
  unsigned char* smem = rmsb_dyn_smem + ((1024u - (smem_u32(rmsb_dyn_smem) & 1023u)) & 1023u);
  FewBars* bars = reinterpret_cast<FewBars*>(smem + pl.ring_bytes);
  float* row_scales = reinterpret_cast<float*>(bars + 1);  // [2][kFewChunk][T]: of the rows of a
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = static_cast<int>(blockIdx.x % pl.splits);
  const int64_t tile = blockIdx.x / pl.splits;
  const int tn = static_cast<int>(tile % pl.tiles_n);
  const int64_t t0 = tile / pl.tiles_n * T;  // first row of a
  const int g0 = static_cast<int>(static_cast<int64_t>(p.groups) * rank / pl.splits);
  const int g1 = static_cast<int>(static_cast<int64_t>(p.groups) * (rank + 1) / pl.splits);
  if (threadIdx.x == 0) {
    for (int i = 0; i < pl.stages; ++i) {
      mbar_init(&bars->full[i], 1);
      mbar_init(&bars->empty[i], 1);
    }
    for (int i = 0; i < F::kSums; ++i) {
      mbar_init(&bars->sum[i], 1);
      mbar_init(&bars->sum_empty[i], 4);
    }
    mbar_init(&bars->done, 1);
    fence_mbar_init();
  }
  if (warp == 5) tmem_alloc_warp(&bars->tmem, F::kTmem);
  if (threadIdx.x == 128) {
    prefetch_map(&map_a);
    prefetch_map(&map_b);
  }
  tmem_fence_before_sync();
  __syncthreads();
  tmem_fence_after_sync();
  const uint32_t tmem = bars->tmem;
  pdl_launch_dependents();  // they may take tensor memory and wait: this grid has all of its own by now
  pdl_wait();

  float2 acc[T / 2];
  const int64_t n = static_cast<int64_t>(tn) * kBlock + threadIdx.x;  // warps 0 - 3: this thread's row of b
  if (warp == 4) {
    int st = 0;
    uint32_t pass = 0;
    for (int g = g0; g < g1; ++g) {
      const bool ok = __all_sync(0xffffffffu, mbar_spin_warp(&bars->empty[st], pass ^ 1u, kSiteMmEmpty));
      if (!ok) break;
      if (elect_one()) {
        unsigned char* at = smem + st * F::kStageBytes;
        mbar_arrive_expect_tx(&bars->full[st], F::kStageBytes);
        tile_load<false>(at, &map_b, g * kTileK, tn * kBlock, &bars->full[st]);
        tile_load<false>(at + kTileBytes, &map_a, g * kTileK, static_cast<int>(t0), &bars->full[st]);
      }
      __syncwarp();
      if (++st == pl.stages) {
        st = 0;
        pass ^= 1u;
      }
    }
    if (lane == 0 && abort_requested())
      for (int i = 0; i < pl.stages; ++i) mbar_wait(&bars->full[i], i < st ? pass : pass ^ 1u, kSiteDrain, false);
    for (int i = 0; i < pl.stages; ++i) mbar_spin_warp(&bars->empty[i], i < st ? pass : pass ^ 1u, kSiteMmEmpty);
  } else if (warp == 5) {
    constexpr uint32_t idesc = product_desc(kBlock, T);
    int st = 0;
    uint32_t pass = 0, u = 0;
    for (int g = g0; g < g1; ++g, ++u) {
      const uint32_t d = u % F::kSums;
      bool ok = mbar_spin_warp(&bars->full[st], pass, kSiteMmFull);
      ok = mbar_spin_warp(&bars->sum_empty[d], ((u / F::kSums) & 1u) ^ 1u, kSiteMmSumEmpty) && ok;
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tmem_fence_after_sync();
      if (elect_one()) {
        const uint32_t at = smem_u32(smem + st * F::kStageBytes);
        const uint64_t a = operand_desc(at), b = operand_desc(at + kTileBytes);
#pragma unroll
        for (int k = 0; k < kTileK / 32; ++k) mma_e4m3<false>(tmem + d * T, a + 2 * k, b + 2 * k, idesc, k > 0);
        mma_commit<false>(&bars->empty[st]);
        mma_commit<false>(&bars->sum[d]);
      }
      __syncwarp();
      if (++st == pl.stages) {
        st = 0;
        pass ^= 1u;
      }
    }
    if (__any_sync(0xffffffffu, abort_requested())) {  // the products issued so far end first
      if (elect_one()) mma_commit<false>(&bars->done);
      __syncwarp();
      if (lane == 0) mbar_wait(&bars->done, 0, kSiteDrain, false);
      __syncwarp();
    }
  } else {
    const uint32_t from = tmem + (static_cast<uint32_t>(warp) << 21);
    const bool b_live = n < p.n;
    const float* sb = sb_of(p, n) + g0 * p.sb_group;
    auto next_b = [&](int g) {
      const float v = b_live && g < g1 ? ld1(sb) : 0.f;
      sb += p.sb_group;
      return v;
    };
    float b0 = next_b(g0), b1 = next_b(g0 + 1);  // two groups ahead
#pragma unroll
    for (int i = 0; i < T / 2; ++i) acc[i] = make_float2(0.f, 0.f);
    // a's scales, kFewChunk groups of T rows at a time, a chunk ahead in registers: thread i has
    // row i % T of groups i / T, i / T + 128 / T, ...
    float ahead[kFewChunk * T / 128];
    auto fetch = [&](int c0) {
#pragma unroll
      for (int j = 0; j < kFewChunk * T / 128; ++j) {
        const int i = threadIdx.x + j * 128, g = c0 + i / T;
        const int64_t t = t0 + i % T;
        ahead[j] = g < g1 && t < p.m ? ld1(p.sa + t * p.sa_row + g * p.sa_group) : 0.f;
      }
    };
    fetch(g0);
    int d = 0, buffer = 0;
    uint32_t pass = 0;
    for (int c0 = g0; c0 < g1; c0 += kFewChunk, buffer ^= 1) {
      const int c1 = min(c0 + kFewChunk, g1);
      float* scales = row_scales + buffer * (kFewChunk * T);
#pragma unroll
      for (int j = 0; j < kFewChunk * T / 128; ++j) scales[threadIdx.x + j * 128] = ahead[j];
      fetch(c0 + kFewChunk);
      __syncwarp();
      named_barrier(1, 128);
      for (int g = c0; g < c1; ++g) {
        const float s = b0;
        const float* rows = scales + (g - c0) * T;
        b0 = b1;
        b1 = next_b(g + 2);
        mbar_spin_warp(&bars->sum[d], pass, kSiteMmSum);
        __syncwarp();
        tmem_fence_after_sync();
        float2 v[T > 64 ? 1 : T / kChunk][kChunk / 2];
        if constexpr (T <= 64) {
#pragma unroll
          for (int c = 0; c < T / kChunk; ++c) tmem_ld(from + d * T + c * kChunk, v[c]);
#pragma unroll
          for (int c = 0; c < T / kChunk; ++c) tmem_landed(v[c]);
        }
#pragma unroll
        for (int c = 0; c < T / kChunk; ++c) {
          float2(&x)[kChunk / 2] = v[T > 64 ? 0 : c];
          if constexpr (T > 64) {
            tmem_ld(from + d * T + c * kChunk, x);
            tmem_landed(x);
          }
          if (c == (T > 64 ? T / kChunk - 1 : 0)) {
            tmem_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->sum_empty[d]);
          }
#pragma unroll
          for (int i = 0; i < kChunk / 2; i += 2) {
            const float4 r = *reinterpret_cast<const float4*>(rows + c * kChunk + 2 * i);
            float2* to = acc + c * (kChunk / 2) + i;
            to[0] = fma2(x[i], mul2(make_float2(r.x, r.y), splat2(s)), to[0]);
            to[1] = fma2(x[i + 1], mul2(make_float2(r.z, r.w), splat2(s)), to[1]);
          }
        }
        if (++d == F::kSums) {
          d = 0;
          pass ^= 1u;
        }
      }
    }
    const float bias = p.bias && b_live ? load1_rt(p.bias, p.bias_dt, n) : 0.f;
    if (pl.splits == 1) {
      if (b_live) {
#pragma unroll
        for (int i = 0; i < T; ++i)
          if (t0 + i < p.m)
            store1_rt(p.out, p.out_dt, (t0 + i) * p.n + n, (i & 1 ? acc[i / 2].y : acc[i / 2].x) + bias);
      }
    } else {
      // every copy has landed and been read: the stages take the sums
      float* part = reinterpret_cast<float*>(smem);  // [T][128]
#pragma unroll
      for (int i = 0; i < T; ++i) part[i * kBlock + threadIdx.x] = i & 1 ? acc[i / 2].y : acc[i / 2].x;
    }
  }
  // Tensor memory goes back before the CTAs of a cluster wait for one another: a peer that has
  // none yet may wait for this CTA's SM.
  __syncwarp();
  tmem_fence_before_sync();
  __syncthreads();
  tmem_fence_after_sync();
  if (warp == 5) tmem_dealloc_warp(tmem, F::kTmem);
  if (pl.splits == 1) return;
  cluster_sync_all();
  // Row i of the result is CTA i % splits's, a warp a row, four columns a lane; the partial sums
  // are added in the order of the CTAs.
  for (int i = rank + warp * pl.splits; i < T && t0 + i < p.m; i += kFewThreads / 32 * pl.splits) {
    const uint32_t at = smem_u32(smem) + static_cast<uint32_t>(i * kBlock + lane * 4) * 4;
    float4 part[kFewMaxSplits];
#pragma unroll
    for (int r = 0; r < kFewMaxSplits; ++r) part[r] = r < pl.splits ? ld_peer4(map_peer(at, r)) : make_float4(0.f, 0.f, 0.f, 0.f);
    float4 sum = part[0];
#pragma unroll
    for (int r = 1; r < kFewMaxSplits; ++r) {
      sum.x += part[r].x; sum.y += part[r].y; sum.z += part[r].z; sum.w += part[r].w;
    }
    const int64_t col = static_cast<int64_t>(tn) * kBlock + lane * 4;
    const float out[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (col + k < p.n)
        store1_rt(p.out, p.out_dt, (t0 + i) * p.n + col + k, out[k] + (p.bias ? load1_rt(p.bias, p.bias_dt, col + k) : 0.f));
  }
  cluster_sync_all();
}

// ---------------------------------------------------------------------------------------
// Operands whose address or row stride is no multiple of 16 (blockIdx.y: one or both), copied to where they are: 16
// bytes a thread from the aligned words around them.
// ---------------------------------------------------------------------------------------
struct RepackJob {
  const unsigned char* src;
  int64_t src_row, rows;
  unsigned char* dst;
};
struct RepackParams {
  RepackJob job[2];
  int32_t k, pieces;  // bytes of a row; pieces of 16 bytes of a row of the copy
};

__global__ void __launch_bounds__(256) repack_kernel(const RepackParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const RepackJob& jb = blockIdx.y == 0 ? p.job[0] : p.job[1];
  const int32_t k = p.k, pieces = p.pieces;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t row = i / pieces;
  if (row >= jb.rows) return;
  const int at = static_cast<int>(i - row * pieces) * 16;
  const unsigned char* s = jb.src + row * jb.src_row + at;
  const int left = min(16, k - at);
  uint32_t w[4] = {0, 0, 0, 0};
  if (left == 16) {
    const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(s)) & 3u;
    const uint32_t* words = reinterpret_cast<const uint32_t*>(s - off);
    uint32_t v[5];
    // the first and last words hold bytes of other rows or of nothing: only those with bytes of
    // this piece are read
#pragma unroll
    for (int j = 0; j < 5; ++j) v[j] = j < 4 || off ? words[j] : 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = __funnelshift_r(v[j], v[j + 1], off * 8);
  } else {
    for (int j = 0; j < left; ++j) {
      const uint32_t b = static_cast<uint32_t>(ld1(s + j)) << (8 * (j & 3));
      if (j < 4) w[0] |= b;
      else if (j < 8) w[1] |= b;
      else if (j < 12) w[2] |= b;
      else w[3] |= b;
    }
  }
  uint4* to = reinterpret_cast<uint4*>(jb.dst) + i;
  if (RMSB_DBG_OK(to, 16, kDbgVecStore)) *to = make_uint4(w[0], w[1], w[2], w[3]);
}

}  // namespace rmsb200
