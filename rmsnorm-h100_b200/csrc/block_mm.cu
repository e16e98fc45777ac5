// block_mm.cu -- rmsnorm_b200_block_mm: argument checks, choice of the kernel and launch.
#define RMSB_UNIT block_mm
#include "unit_state.cuh"

#include "block_mm_kernels.cuh"

namespace rmsb200 {
namespace {

using FewKernel = void (*)(const CUtensorMap, const CUtensorMap, const BlockMmParams, const FewPlan);
using WideKernel = void (*)(const CUtensorMap, const CUtensorMap, const BlockMmParams, const WidePlan);
using EncodeTiled = decltype(&cuTensorMapEncodeTiled);

// The driver's function that makes tensor maps (the library does not link the driver).
EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      p = nullptr;
    cudaGetLastError();
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

// Boxes of `box_rows` rows and kTileK bytes of a byte matrix.
int make_map(CUtensorMap* map, const void* base, int64_t rows, int64_t k, int64_t row_stride, int box_rows) {
  const EncodeTiled encode = encode_tiled();
  if (!encode) return RMSNORM_B200_ERR_CUDA;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(row_stride)};
  const cuuint32_t box[2] = {kTileK, static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t each[2] = {1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, each,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? RMSNORM_B200_OK
             : RMSNORM_B200_ERR_CUDA;
}

// TMA reads operands at addresses and row strides that are multiples of 16.
bool tma_ready(const void* base, int64_t rows, int64_t row_stride) {
  return aligned_to(base, 16) && (row_stride % 16 == 0 || rows == 1);
}

struct Plan {
  int64_t pitch = 0;  // row stride of the copies
  size_t copy_a = 0, copy_b = 0;
};

int check(const rmsnorm_b200_block_mm_args* a) {
  constexpr int64_t kMost = int64_t{1} << 31;
  if (!a || a->m < 0 || a->n < 1 || a->k < 1 || a->m >= kMost || a->n >= kMost || a->k >= kMost)
    return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if ((a->b_block_rows != 1 && a->b_block_rows != kBlock) || !valid_dt(a->out_dtype) ||
      (a->bias && !valid_dt(a->bias_dtype)))
    return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (a->m == 0) return RMSNORM_B200_OK;
  if (!a->a || !a->b || !a->a_scales || !a->b_scales || !a->out) return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (a->a_row_stride < 0 || a->b_row_stride < 0 || a->a_scale_row_stride < 0 || a->a_scale_group_stride < 0 ||
      a->b_scale_row_stride < 0 || a->b_scale_group_stride < 0)
    return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if ((a->m > 1 && a->a_row_stride < a->k) || (a->n > 1 && a->b_row_stride < a->k))
    return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  return RMSNORM_B200_OK;
}

Plan make_plan(const rmsnorm_b200_block_mm_args* a) {
  Plan pl;
  pl.pitch = (a->k + 15) / 16 * 16;
  if (!tma_ready(a->a, a->m, a->a_row_stride)) pl.copy_a = static_cast<size_t>(a->m) * pl.pitch;
  if (!tma_ready(a->b, a->n, a->b_row_stride)) pl.copy_b = static_cast<size_t>(a->n) * pl.pitch;
  return pl;
}

struct MmLaunch {
  const char* kind;
  unsigned grid;
  int tile, splits, stages;
};

std::string describe(const void* data) {
  const MmLaunch& l = *static_cast<const MmLaunch*>(data);
  char buf[128];
  std::snprintf(buf, sizeof(buf), "%s grid=%u tile=%d splits=%d stages=%d", l.kind, l.grid, l.tile, l.splits, l.stages);
  return buf;
}

// Called with the device's lock held.
template <typename Kernel>
int prepare(UnitDevice* ud, Kernel kernel) {
  const void* fn = reinterpret_cast<const void*>(kernel);
  if (ud->attrs_done.count(fn)) return RMSNORM_B200_OK;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemOptIn) != cudaSuccess)
    return RMSNORM_B200_ERR_CUDA;
  ud->attrs_done.insert(fn);
  return RMSNORM_B200_OK;
}

template <typename Kernel, typename KernelPlan>
int launch(UnitDevice* ud, Kernel kernel, const CUtensorMap& ma, const CUtensorMap& mb, const BlockMmParams& p,
           const KernelPlan& kp, int threads, int smem, int cluster, cudaStream_t stream, const MmLaunch& l) {
  {
    std::lock_guard<std::mutex> lock(ud->mu);
    const int st = prepare(ud, kernel);
    if (st) return st;
  }
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(l.grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, kernel, ma, mb, p, kp) != cudaSuccess) {
    cudaGetLastError();
    return RMSNORM_B200_ERR_CUDA;
  }
  return launched(describe, l);
}

int repack(const RepackJob* jobs, int count, int64_t k, int64_t pitch, cudaStream_t stream) {
  RepackParams p = {};
  int64_t rows = 0;
  for (int i = 0; i < count; ++i) {
    p.job[i] = jobs[i];
    rows = std::max(rows, jobs[i].rows);
  }
  p.k = static_cast<int32_t>(k);
  p.pieces = static_cast<int32_t>(pitch / 16);
  if (rows > (int64_t{1} << 38) / p.pieces) return RMSNORM_B200_ERR_UNSUPPORTED;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((rows * p.pieces + 255) / 256), count);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, repack_kernel, p) != cudaSuccess) {
    cudaGetLastError();
    return RMSNORM_B200_ERR_CUDA;
  }
  return launched("");
}

// Clusters of the kernel with `cluster` CTAs that are resident together, a CTA an SM.
template <typename Kernel>
int resident(UnitDevice* ud, Kernel kernel, int threads, int cluster, int smem, int* clusters) {
  const void* fn = reinterpret_cast<const void*>(kernel);
  std::lock_guard<std::mutex> lock(ud->mu);
  const auto key = std::make_tuple(fn, cluster, smem);
  const auto it = ud->clusters.find(key);
  if (it != ud->clusters.end()) {
    *clusters = it->second;
    return RMSNORM_B200_OK;
  }
  const int st = prepare(ud, kernel);
  if (st) return st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(cluster * ud->sm_count);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(clusters, kernel, &cfg) != cudaSuccess) *clusters = 0;
  cudaGetLastError();
  ud->clusters[key] = *clusters;
  return RMSNORM_B200_OK;
}

template <int T>
int launch_few(UnitDevice* ud, const void* a, int64_t a_row, const CUtensorMap& map_b, const rmsnorm_b200_block_mm_args* args,
               const BlockMmParams& p, cudaStream_t stream) {
  CUtensorMap map_a;
  int st = make_map(&map_a, a, args->m, args->k, a_row, T);
  if (st) return st;
  FewPlan pl = {};
  pl.tiles_n = static_cast<int>((args->n + kBlock - 1) / kBlock);
  const int64_t tiles = (args->m + T - 1) / T * pl.tiles_n;
  constexpr int fit = T >= 128 ? 1 : 2;  // CTAs an SM
  // As many parts as are resident together, of two groups at least: 1 x 4096 x 4096 in 1, 2, 4, 6
  // and 8 parts 11.5, 8.6, 7.7, 7.0 and 6.7 us, 64 x 8192 x 8192 38, 24, 17.3, 24 and 25 us,
  // 32 x 4096 x 1024 6.8, 5.1, 5.2, -- and (a group each) 6.2 us, 256 x 1024 x 4096 22.6, 12.9, 9.2,
  // 8.6 and 14.2 us (16 clusters of 8: 15 fit at once).
  pl.splits = static_cast<int>(std::clamp<int64_t>(fit * ud->sm_count / tiles, 1, std::clamp(p.groups / 2, 1, kFewMaxSplits)));
  int smem = 0;
  for (;; --pl.splits) {
    const int each = (p.groups + pl.splits - 1) / pl.splits;
    const int fixed = 1024 + static_cast<int>(sizeof(FewBars)) + 2 * kFewChunk * T * 4;
    const int room = (fit == 2 ? kSmemOptIn / 2 - 1024 : kSmemOptIn) - fixed;
    pl.stages = std::min({kFewMaxStages, each, room / Few<T>::kStageBytes});
    pl.ring_bytes = std::max(pl.stages * Few<T>::kStageBytes, pl.splits > 1 ? T * kBlock * 4 : 0);
    smem = pl.ring_bytes + fixed;
    if (pl.splits == 1) break;
    int clusters = 0;
    st = resident<FewKernel>(ud, block_mm_few_kernel<T>, kFewThreads, pl.splits, smem, &clusters);
    if (st) return st;
    if (clusters * fit >= tiles) break;
  }
  if (tiles * pl.splits >= int64_t{1} << 31) return RMSNORM_B200_ERR_UNSUPPORTED;
  const MmLaunch l = {"block_mm_few", static_cast<unsigned>(tiles * pl.splits), T, pl.splits, pl.stages};
  return launch<FewKernel>(ud, block_mm_few_kernel<T>, map_a, map_b, p, pl, kFewThreads, smem, pl.splits, stream, l);
}

// Pairs of CTAs, one tile after the other.
int launch_pairs(UnitDevice* ud, const char* kind, WideKernel kernel, int threads, int tile_n, int stages, int smem,
                 const CUtensorMap& map_a, const CUtensorMap& map_b, const rmsnorm_b200_block_mm_args* a,
                 const BlockMmParams& p, cudaStream_t stream) {
  WidePlan pl = {};
  pl.tiles_m = static_cast<int>((a->m + kWideRows - 1) / kWideRows);
  pl.tiles_n = static_cast<int>((a->n + tile_n - 1) / tile_n);
  pl.band = 12;  // 8 to 16 within 2 % of one another, 4 and 32 6 and 12 % slower (8192 x 16384 x 4096)
  const int64_t tiles = static_cast<int64_t>(pl.tiles_m) * pl.tiles_n;
  const int64_t pairs = std::min<int64_t>(tiles, ud->sm_count / 2);
  const MmLaunch l = {kind, static_cast<unsigned>(pairs * 2), tile_n, 1, stages};
  return launch<WideKernel>(ud, kernel, map_a, map_b, p, pl, threads, smem, 2, stream, l);
}

template <int N>
int launch_scaled(UnitDevice* ud, const CUtensorMap& map_a, const void* b, int64_t b_row,
                  const rmsnorm_b200_block_mm_args* args, const BlockMmParams& p, cudaStream_t stream) {
  constexpr int kSmem = 1024 + kScaledStages * (ScaledTile<N>::kStageBytes + kExpBytes) + static_cast<int>(sizeof(ScaledBars)) +
                        8 * kStagingBytes;
  static_assert(kSmem <= kSmemOptIn, "shared memory");
  CUtensorMap map_b;
  const int st = make_map(&map_b, b, args->n, args->k, b_row, N / 2);
  if (st) return st;
  return launch_pairs(ud, "block_mm_scaled", block_mm_scaled_kernel<N>, kScaledThreads, N, kScaledStages, kSmem, map_a, map_b,
                      args, p, stream);
}

int launch_wide(UnitDevice* ud, const void* a, int64_t a_row, const void* b, int64_t b_row,
                const rmsnorm_b200_block_mm_args* args, const BlockMmParams& p, cudaStream_t stream) {
  constexpr int kSmem = 1024 + kWideStages * kWideStageBytes + static_cast<int>(sizeof(WideBars)) + 2 * kWideN * 4 +
                        8 * kStagingBytes;
  static_assert(kSmem <= kSmemOptIn, "shared memory");
  CUtensorMap map_a, map_b;
  int st = make_map(&map_a, a, args->m, args->k, a_row, kBlock);
  if (st) return st;
  if (args->power_of_two && args->out_dtype != RMSNORM_B200_F32) {
    // The width of a tile that leaves the least to do one after the other: rounds of tiles, each of
    // N columns a group, and for the widest the time its results take to come out (about 1600
    // cycles, of which a column takes two a group). fp32 results keep the sum of the groups' sums
    // in registers, whose additions round to nearest.
    const int64_t pairs = ud->sm_count / 2, tiles_m = (args->m + kWideRows - 1) / kWideRows;
    auto cost = [&](int64_t n, int64_t alone) {
      return (tiles_m * ((args->n + n - 1) / n) + pairs - 1) / pairs * (p.groups * n + alone);
    };
    const int64_t c256 = cost(256, 800), c224 = cost(224, 0), c192 = cost(192, 0);
    if (c224 <= c256 && c224 <= c192) return launch_scaled<224>(ud, map_a, b, b_row, args, p, stream);
    if (c192 <= c256) return launch_scaled<192>(ud, map_a, b, b_row, args, p, stream);
    return launch_scaled<256>(ud, map_a, b, b_row, args, p, stream);
  }
  st = make_map(&map_b, b, args->n, args->k, b_row, kBlock);
  if (st) return st;
  return launch_pairs(ud, "block_mm_wide", p.b_rows ? block_mm_wide_kernel<true> : block_mm_wide_kernel<false>, kWideThreads,
                      kWideN, kWideStages, kSmem, map_a, map_b, args, p, stream);
}

int run(const rmsnorm_b200_block_mm_args* a, void* ws, size_t ws_bytes, cudaStream_t stream) {
  int st = check(a);
  if (st) return st;
  if (a->m == 0) {
    rmsb_units::set_last_plan("block_mm empty");
    return RMSNORM_B200_OK;
  }
  UnitDevice* ud = nullptr;
  st = unit_device(&ud);
  if (st) return st;
  const Plan pl = make_plan(a);
  const size_t need = pl.copy_a + pl.copy_b;
  if (need > ws_bytes || (need > 0 && (!ws || !aligned_to(ws, 16)))) return RMSNORM_B200_ERR_WORKSPACE;
  const int64_t groups = (a->k + kBlock - 1) / kBlock;
  Ranges ranges;
  ranges.add(a->a, (a->m - 1) * a->a_row_stride + a->k);
  ranges.add(a->b, (a->n - 1) * a->b_row_stride + a->k);
  ranges.add(a->a_scales, ((a->m - 1) * a->a_scale_row_stride + (groups - 1) * a->a_scale_group_stride + 1) * 4);
  const int64_t b_rows = (a->n + a->b_block_rows - 1) / a->b_block_rows;
  ranges.add(a->b_scales, ((b_rows - 1) * a->b_scale_row_stride + (groups - 1) * a->b_scale_group_stride + 1) * 4);
  if (a->bias) ranges.add(a->bias, a->n * elem_bytes(a->bias_dtype));
  ranges.add_out(a->out, static_cast<size_t>(a->m) * a->n * elem_bytes(a->out_dtype));
  ranges.add(ws, need);
  st = ranges.send(stream);
  if (st) return st;

  const void *qa = a->a, *qb = a->b;
  int64_t a_row = a->m == 1 ? pl.pitch : a->a_row_stride, b_row = a->n == 1 ? pl.pitch : a->b_row_stride;
  RepackJob jobs[2];
  int copies = 0;
  if (pl.copy_a) {
    jobs[copies++] = {static_cast<const unsigned char*>(a->a), a->a_row_stride, a->m, static_cast<unsigned char*>(ws)};
    qa = ws;
    a_row = pl.pitch;
  }
  if (pl.copy_b) {
    unsigned char* to = static_cast<unsigned char*>(ws) + pl.copy_a;
    jobs[copies++] = {static_cast<const unsigned char*>(a->b), a->b_row_stride, a->n, to};
    qb = to;
    b_row = pl.pitch;
  }
  if (copies) {
    st = repack(jobs, copies, a->k, pl.pitch, stream);
    if (st) return st;
  }
  BlockMmParams p = {};
  p.m = a->m; p.n = static_cast<int32_t>(a->n); p.groups = static_cast<int32_t>(groups);
  p.sa = a->a_scales; p.sa_row = a->a_scale_row_stride; p.sa_group = a->a_scale_group_stride;
  p.sb = a->b_scales; p.sb_row = a->b_scale_row_stride; p.sb_group = a->b_scale_group_stride;
  p.bias = a->bias; p.bias_dt = a->bias_dtype;
  p.out = a->out; p.out_dt = a->out_dtype;
  p.b_rows = a->b_block_rows == 1;
  p.vec_bias = aligned_to(a->bias, 16);
  p.vec_out = aligned_to(a->out, 32) && a->n * elem_bytes(a->out_dtype) % 32 == 0;
  // Few rows, or more of them where two CTAs or more could share each 128 x 128 of the result:
  // the kernel that splits k. K = 4096: 256 x 4096 14.4 against 20.1 us, 1024 x 1024 14.2 against
  // 20.0 us, 512 x 4096 (128 tiles for 148 SMs) 24.8 against 20.3 us.
  const int64_t squares = (a->m + kBlock - 1) / kBlock * ((a->n + kBlock - 1) / kBlock);
  if (a->m > 128 && (2 * squares > ud->sm_count || groups < 4)) return launch_wide(ud, qa, a_row, qb, b_row, a, p, stream);
  CUtensorMap map_b;
  st = make_map(&map_b, qb, a->n, a->k, b_row, kBlock);
  if (st) return st;
  if (a->m <= 16) return launch_few<16>(ud, qa, a_row, map_b, a, p, stream);
  if (a->m <= 32) return launch_few<32>(ud, qa, a_row, map_b, a, p, stream);
  if (a->m <= 64) return launch_few<64>(ud, qa, a_row, map_b, a, p, stream);
  return launch_few<128>(ud, qa, a_row, map_b, a, p, stream);
}

int workspace_size(const rmsnorm_b200_block_mm_args* a, size_t* bytes) {
  if (!bytes) return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  *bytes = 0;
  const int st = check(a);
  if (st || a->m == 0) return st;
  const Plan pl = make_plan(a);
  *bytes = pl.copy_a + pl.copy_b;
  return RMSNORM_B200_OK;
}

}  // namespace
}  // namespace rmsb200

using namespace rmsb200;

extern "C" int rmsnorm_b200_block_mm_workspace_size(const rmsnorm_b200_block_mm_args* a, size_t* bytes) {
  return entry([&] { return workspace_size(a, bytes); });
}

extern "C" int rmsnorm_b200_block_mm(const rmsnorm_b200_block_mm_args* a, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  return entry([&] { return run(a, workspace, workspace_bytes, static_cast<cudaStream_t>(stream)); });
}
