// row_plan.h -- launch plan of the fused row kernels (row_ring.cuh has the vocabulary).
#pragma once

#include <cstring>

#include "row_ring.cuh"

namespace rmsb200 {
namespace {

inline int pow2_ceil(int64_t v) {
  int p = 1;
  while (p < v) p <<= 1;
  return p;
}

constexpr int kRingBytes = 200 * 1024;  // of shared memory, for two whole rows of every group

// What a kernel asks of its plan.
struct RowWants {
  bool odd = false;      // the kernels of odd_kernels.cuh; otherwise N is a multiple of 8
  int built_in = 0;      // row group of a kernel made for one: four steps, units of bwd_unit_steps, a row each
  bool shifted = false;  // units of one row; one step or max_steps
  int scale = 0;         // columns of a scale whose largest value passes through shared memory
  bool whole = false;    // a row's slice is one unit; two of them a group
};

// Columns of a row of N on shifted vectors (shift_rows.cuh), whatever its lead.
inline int64_t shifted_columns(int64_t N) {
  const int64_t most = N % 2 ? 7 : N % 4 ? 6 : N % 8 ? 4 : 0;
  return (N + most + 7) / 8 * 8;
}

// Plans rows of N columns whose tensors have elements of bytes[i] (0: absent); threads of a CTA,
// max_steps: vector steps a thread can hold. Returns why there is no plan, or null.
inline const char* plan_rows(int64_t rows, int64_t N, const int (&bytes)[3], bool bias, int threads, int max_steps,
                             int sms, RowPlan* pl, int* k, int* smem, const RowWants& want = {}) {
  const bool odd = want.odd;
  const int built_in = want.built_in;
  const int64_t cta_cols = static_cast<int64_t>(threads) * 8 * max_steps;
  if (N > cta_cols * kMaxRowCtas) return "rows wider than a cluster holds";
  pl->C = N > cta_cols ? pow2_ceil((N + cta_cols - 1) / cta_cols) : 1;
  pl->slice = static_cast<int>(N);
  if (pl->C > 1) {
    const int64_t per = (N + pl->C - 1) / pl->C;
    pl->slice = static_cast<int>((per + kScaleAlign - 1) / kScaleAlign * kScaleAlign);
  }
  const int vecs = (pl->slice + 7) / 8;
  // Few rows: as many threads to a row as it has vectors, for the latency. Otherwise as few as
  // hold it, so that a CTA works on several rows at once and their totals overlap.
  const int steps = rows <= sms ? 1 : max_steps;
  const int per_row = (vecs + steps - 1) / steps;
  const int elem = bytes[0] + bytes[1] + bytes[2];
  if (built_in) {
    pl->G = built_in;
    pl->groups = pl->C > 1 ? 1 : threads / pl->G;
  } else if (odd || rows <= sms) {
    pl->G = std::clamp(pow2_ceil(per_row), 32, threads);
    pl->groups = pl->C > 1 ? 1 : threads / pl->G;
  } else {
    // as many groups as their rows' vectors allow, of any number of warps, the steps shared out
    // evenly: 2368 columns in five groups of 96 threads 247 us, in four of 128 301 us (5.7e4 rows, bf16)
    pl->groups = pl->C > 1 ? 1 : threads / std::clamp((per_row + 31) / 32 * 32, 32, threads);
    while (want.whole && pl->groups > 1 && 2 * pl->groups * vecs * 8 * elem > kRingBytes) --pl->groups;
    const int most = threads / pl->groups / 32 * 32, used = (vecs + most - 1) / most;
    pl->G = ((vecs + used - 1) / used + 31) / 32 * 32;
  }
  *k = built_in ? max_steps : pow2_ceil((vecs + pl->G - 1) / pl->G);
  if (want.shifted && *k > 1) *k = max_steps;
  // Units of up to 32 KB: larger ones leave too few in flight (32768 x 16384 bf16 + residual,
  // fp32 residual_out, 8 bits: 748 us in five units of 32 KB, 842 us in two of 64 KB).
  pl->KC = *k;
  while (!want.whole && pl->KC > 1 && pl->KC * pl->G * 8 * elem > 32768) pl->KC >>= 1;
  if (built_in) pl->KC = bwd_unit_steps(built_in);
  pl->unit_shift = 0;
  while ((pl->KC << pl->unit_shift) < *k) ++pl->unit_shift;
  // Short rows go several to a unit: a copy of about 4 KB at least, but no fewer tiles than groups.
  pl->R = 1;
  if (pl->C == 1 && pl->KC == *k && !built_in && !want.shifted) {
    const int64_t fair = rows / (static_cast<int64_t>(sms) * pl->groups);
    pl->R = static_cast<int>(std::clamp<int64_t>(std::min<int64_t>(4096 / (N * elem), fair), 1, 8));
  }
  const int unit_cols = pl->R > 1 ? pl->R * pl->slice : std::min(pl->slice, pl->KC * pl->G * 8);
  uint32_t off = 0;
  for (int i = 0; i < 3; ++i) {
    pl->off[i] = off;
    // odd rows: up to 15 bytes before the first element, and up to the end of its last granule
    if (bytes[i]) off += odd ? (unit_cols * bytes[i] + 45) & ~15 : unit_cols * bytes[i];
  }
  pl->unit_bytes = (off + 127u) & ~127u;
  pl->bias = bias;
  pl->tiles = (rows + pl->R - 1) / pl->R;
  if (odd) pl->slice = (pl->slice + 7) & ~7;  // the affine copies keep the barriers' alignment
  const int affine = pl->slice * 4 * (bias ? 2 : 1);
  pl->scale_slots = want.scale ? pl->slice / want.scale + 1 : 0;
  const int fixed = affine + static_cast<int>(sizeof(RowBars)) + 8 * pl->scale_slots * pl->groups + 16;
  const int unit = pl->groups * static_cast<int>(pl->unit_bytes);
  const int64_t per_group = (pl->tiles * pl->C + static_cast<int64_t>(sms) * pl->groups - 1) /
                            (static_cast<int64_t>(sms) * pl->groups);
  pl->S = std::min({16, kMaxUnits / pl->groups, (kSmemOptIn - fixed) / unit});
  pl->S = static_cast<int>(std::min<int64_t>(pl->S, std::max<int64_t>(1, per_group << pl->unit_shift)));
  if (pl->S < 1) return "rows too wide for shared memory";
  *smem = pl->S * unit + fixed;
  return nullptr;
}

struct RowLaunch {  // for rmsnorm_b200_last_plan
  RowPlan pl;
  char kind[16];
  int grid, k, smem;
};

inline std::string describe_rows(const void* data) {
  const RowLaunch& l = *static_cast<const RowLaunch*>(data);
  char buf[192];
  std::snprintf(buf, sizeof(buf), "%s grid=%d G=%d groups=%d K=%d KC=%d R=%d S=%d C=%d slice=%d unit=%u smem=%d", l.kind,
                l.grid, l.pl.G, l.pl.groups, l.k, l.pl.KC, l.pl.R, l.pl.S, l.pl.C, l.pl.slice, l.pl.unit_bytes, l.smem);
  return buf;
}

// Clusters of the plan's shape (CTAs, without a split) that can be resident at once.
template <typename Kernel>
int resident_clusters(UnitDevice* ud, Kernel kernel, const RowPlan& pl, int smem, int* clusters) {
  const void* fn = reinterpret_cast<const void*>(kernel);
  std::lock_guard<std::mutex> lock(ud->mu);
  if (!ud->attrs_done.count(fn)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemOptIn) != cudaSuccess ||
        cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
      return RMSNORM_B200_ERR_CUDA;
    ud->attrs_done.insert(fn);
  }
  *clusters = ud->sm_count;
  if (pl.C == 1) return RMSNORM_B200_OK;
  const auto key = std::make_tuple(fn, pl.C, smem);
  const auto it = ud->clusters.find(key);
  if (it != ud->clusters.end()) {
    *clusters = it->second;
    return RMSNORM_B200_OK;
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = pl.C;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(pl.C * ud->sm_count);
  cfg.blockDim = dim3(pl.G * pl.groups);
  cfg.dynamicSmemBytes = smem;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(clusters, kernel, &cfg) != cudaSuccess) *clusters = 0;
  cudaGetLastError();
  ud->clusters[key] = *clusters;
  return RMSNORM_B200_OK;
}

// Launches a persistent grid: one CTA per SM (as many clusters as fit), at most one row group per
// tile. Returns UNSUPPORTED when no cluster of this shape fits.
template <typename Kernel, typename Params>
int launch_rows(UnitDevice* ud, Kernel kernel, const Params& p, const RowPlan& pl, int smem, cudaStream_t stream,
                const char* kind, int k, int* grid_out = nullptr, bool dry_run = false) {
  int clusters = 0;
  const int st = resident_clusters(ud, kernel, pl, smem, &clusters);
  if (st) return st;
  if (clusters < 1) return RMSNORM_B200_ERR_UNSUPPORTED;
  const int64_t grid = std::min<int64_t>(pl.tiles, clusters) * pl.C;
  if (grid_out) *grid_out = static_cast<int>(grid);
  if (dry_run) return RMSNORM_B200_OK;
  cudaLaunchAttribute attr[1];
  if (pl.C > 1) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = pl.C;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
  } else {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(pl.G * pl.groups);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, p, pl) != cudaSuccess) {
    cudaGetLastError();
    return RMSNORM_B200_ERR_CUDA;
  }
  RowLaunch l = {pl, {}, static_cast<int>(grid), k, smem};
  std::strncpy(l.kind, kind, sizeof(l.kind) - 1);
  return launched(describe_rows, l);
}

// The same for kernels on shifted vectors, whose every class of rows needs a cluster.
template <typename Kernel, typename Params>
int launch_shifted(UnitDevice* ud, Kernel kernel, const Params& p, const RowPlan& pl, int smem, cudaStream_t stream,
                   const char* kind, int k, int* grid_out = nullptr, bool dry_run = false) {
  int clusters = 0;
  const int st = resident_clusters(ud, kernel, pl, smem, &clusters);
  if (st) return st;
  if (clusters < 8) return RMSNORM_B200_ERR_UNSUPPORTED;
  return launch_rows(ud, kernel, p, pl, smem, stream, kind, k, grid_out, dry_run);
}

}  // namespace
}  // namespace rmsb200
