// block_quant.cu -- rmsnorm_b200_block_quant: argument checks, plan and launch.
#define RMSB_UNIT block_quant
#include "unit_state.cuh"

#include "block_quant_kernels.cuh"
#include "column_sums.cuh"

namespace rmsb200 {
namespace {

using TileKernel = void (*)(const BlockQuantParams, uint32_t);
using GroupKernel = void (*)(const BlockQuantParams, int64_t, uint32_t);

int64_t blocks_of(int64_t n) { return (n + kBlock - 1) / kBlock; }

int check(const rmsnorm_b200_block_quant_args* a) {
  if (!a || a->rows < 0 || a->cols < 1 || !valid_dt(a->x_dtype)) return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (a->block_rows != 1 && a->block_rows != kBlock) return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (a->column_sums && !valid_dt(a->column_sums_dtype)) return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (a->rows == 0) return RMSNORM_B200_OK;
  if (!a->q && !a->q_t && !a->column_sums) return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (!a->x || (a->q && !a->scales) || (a->q_t && !a->scales_t)) return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (a->x_row_stride < 0 || (a->q && a->q_row_stride < a->cols) || (a->q_t && a->q_t_row_stride < a->rows) ||
      a->scale_row_stride < 0 || a->scale_group_stride < 0)
    return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  // a tile a CTA, or 16 groups
  if (blocks_of(a->rows) > (int64_t{1} << 31) / blocks_of(a->cols) - 1 || a->rows > (int64_t{1} << 33) / blocks_of(a->cols))
    return RMSNORM_B200_ERR_UNSUPPORTED;
  return RMSNORM_B200_OK;
}

bool tiled(const rmsnorm_b200_block_quant_args* a) { return a->block_rows > 1 || a->q_t || a->column_sums; }

size_t workspace(const rmsnorm_b200_block_quant_args* a) {
  return a->column_sums ? static_cast<size_t>(blocks_of(a->rows)) * static_cast<size_t>(a->cols) * sizeof(float) : 0;
}

template <typename X>
TileKernel tiles(int block_rows) {
  return block_rows > 1 ? quant_tiles_kernel<X, true> : quant_tiles_kernel<X, false>;
}

template <typename... Args>
int launch(void (*kernel)(Args...), dim3 grid, int threads, cudaStream_t stream, Args... args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, args...) != cudaSuccess) {
    cudaGetLastError();
    return RMSNORM_B200_ERR_CUDA;
  }
  return RMSNORM_B200_OK;
}

// A grid's text.
struct QuantLaunch {
  char kind[16];
  unsigned grid;
};

std::string describe(const void* data) {
  const QuantLaunch& l = *static_cast<const QuantLaunch*>(data);
  return std::string(l.kind) + " grid=" + std::to_string(l.grid);
}

int run(const rmsnorm_b200_block_quant_args* a, void* ws, size_t ws_bytes, cudaStream_t stream) {
  int st = check(a);
  if (st) return st;
  const size_t need = workspace(a);
  if (need > ws_bytes || (need > 0 && (!ws || !aligned_to(ws, 16)))) return RMSNORM_B200_ERR_WORKSPACE;
  if (a->rows == 0 && !a->column_sums) {
    rmsb_units::set_last_plan("block_quant empty");
    return RMSNORM_B200_OK;
  }
  UnitDevice* ud = nullptr;
  st = unit_device(&ud);
  if (st) return st;
  const int64_t rb = blocks_of(a->rows), cb = blocks_of(a->cols);
  Ranges ranges;
  ranges.add(a->x, a->rows ? ((a->rows - 1) * a->x_row_stride + a->cols) * elem_bytes(a->x_dtype) : 0);
  if (a->q && a->rows) {
    ranges.add_out(a->q, (a->rows - 1) * a->q_row_stride + a->cols);
    const int64_t sr = a->block_rows > 1 ? rb : a->rows;
    ranges.add(a->scales, ((sr - 1) * a->scale_row_stride + (cb - 1) * a->scale_group_stride + 1) * 4);
  }
  if (a->q_t && a->rows) {
    ranges.add(a->q_t, (a->cols - 1) * a->q_t_row_stride + a->rows);
    ranges.add(a->scales_t, (a->block_rows > 1 ? cb : a->cols) * rb * 4);
  }
  if (a->column_sums) ranges.add(a->column_sums, a->cols * elem_bytes(a->column_sums_dtype));
  ranges.add(ws, need);
  st = ranges.send(stream);
  if (st) return st;

  BlockQuantParams p = {};
  p.x = a->x; p.x_row = a->x_row_stride;
  p.q = a->q; p.q_row = a->q_row_stride;
  p.scales = a->scales; p.scale_row = a->scale_row_stride; p.scale_group = a->scale_group_stride;
  p.q_t = a->q_t; p.q_t_row = a->q_t_row_stride; p.scales_t = a->scales_t;
  p.sum_part = a->column_sums ? static_cast<float*>(ws) : nullptr;
  p.rows = a->rows; p.cols = a->cols;
  const int xb = elem_bytes(a->x_dtype);
  p.vec_in = aligned_to(a->x, 16) && a->x_row_stride * xb % 16 == 0;
  p.vec_q = aligned_to(a->q, 8) && a->q_row_stride % 8 == 0;
  p.vec_t = aligned_to(a->q_t, 16) && a->q_t_row_stride % 16 == 0;
  p.vec_all = p.vec_in && (!a->q || p.vec_q) && (!a->q_t || p.vec_t);
  if (a->rows > 0) {
    QuantLaunch l = {};
    // Row groups alone go by tiles where 16-bit values fill three CTAs on every SM: bf16, 8192 x
    // 4096 takes 19.2 us by tiles and 26.1 by groups, 2048 x 4096 6.4 and 7.2, 1024 x 4096 4.5 and
    // 4.2. fp32 gains nothing (2048 x 4096: 9.0 and 7.9, 8192 x 4096: 28.2 and 28.2), and neither
    // do rows without vectors (8192 x 4097: 50.3 and 32.7).
    const bool wide = xb == 2 && p.vec_all && rb * cb >= int64_t{3} * ud->sm_count;
    if (tiled(a) || wide) {
      TileKernel kernel = a->x_dtype == RMSNORM_B200_F32    ? tiles<float>(a->block_rows)
                          : a->x_dtype == RMSNORM_B200_BF16 ? tiles<__nv_bfloat16>(a->block_rows)
                                                            : tiles<__half>(a->block_rows);
      l = {"quant_tiles", static_cast<unsigned>(rb * cb)};
      st = launch(kernel, dim3(l.grid), 256, stream, p, static_cast<uint32_t>(cb));
    } else {
      const int64_t total = a->rows * cb;
      GroupKernel kernel = a->x_dtype == RMSNORM_B200_F32    ? quant_groups_kernel<float>
                           : a->x_dtype == RMSNORM_B200_BF16 ? quant_groups_kernel<__nv_bfloat16>
                                                             : quant_groups_kernel<__half>;
      l = {"quant_groups", static_cast<unsigned>((total + 15) / 16)};
      st = launch(kernel, dim3(l.grid), 256, stream, p, total, static_cast<uint32_t>(cb));
    }
    if (!st) st = launched(describe, l);
    if (st) return st;
  } else {
    rmsb_units::set_last_plan("block_quant empty");
  }
  if (!a->column_sums) return RMSNORM_B200_OK;
  ReduceParams rp = {};
  rp.C = rb;
  rp.W = rp.N = a->cols;
  ReduceJob& jb = rp.job[0];
  jb.part = p.sum_part;
  jb.out = a->column_sums;
  jb.wout = a->cols;
  jb.fold = 1;
  jb.out_dt = a->column_sums_dtype;
  const int64_t cols = reduce_vectorised(jb, rp.W) ? kReduceVCols : kReduceCols;
  reduce_partials_kernel<<<dim3(static_cast<unsigned>((a->cols + cols - 1) / cols)), kReduceThreads, 0, stream>>>(rp);
  return launched("");
}

int workspace_size(const rmsnorm_b200_block_quant_args* a, size_t* bytes) {
  if (!bytes) return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  *bytes = 0;
  const int st = check(a);
  if (st) return st;
  *bytes = workspace(a);
  return RMSNORM_B200_OK;
}

}  // namespace
}  // namespace rmsb200

using namespace rmsb200;

extern "C" int rmsnorm_b200_block_quant_workspace_size(const rmsnorm_b200_block_quant_args* a, size_t* bytes) {
  return entry([&] { return workspace_size(a, bytes); });
}

extern "C" int rmsnorm_b200_block_quant(const rmsnorm_b200_block_quant_args* a, void* workspace,
                                        size_t workspace_bytes, void* stream) {
  return entry([&] { return run(a, workspace, workspace_bytes, static_cast<cudaStream_t>(stream)); });
}
