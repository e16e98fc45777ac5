// fused_fwd.cu -- rmsnorm_b200_quant_fwd and rmsnorm_b200_dropout_rmsnorm_fwd: argument
// checks, plan and launch.
#define RMSB_UNIT fused_fwd
#include "unit_state.cuh"

#include "fused_fwd_kernels.cuh"
#include "row_plan.h"

namespace rmsb200 {
namespace {

using FwdKernel = void (*)(const FusedFwdParams, const RowPlan);
constexpr int kNone = -1;

template <typename X, typename RT>
FwdKernel pick_steps(int k, bool drop) {
  switch (k) {
    case 1: return drop ? fused_fwd_kernel<X, RT, 1, true> : fused_fwd_kernel<X, RT, 1, false>;
    case 2: return drop ? fused_fwd_kernel<X, RT, 2, true> : fused_fwd_kernel<X, RT, 2, false>;
    default: return drop ? fused_fwd_kernel<X, RT, 4, true> : fused_fwd_kernel<X, RT, 4, false>;
  }
}

FwdKernel pick(int x, int res, int k, bool drop) {
  constexpr int H = RMSNORM_B200_F16, B = RMSNORM_B200_BF16, F = RMSNORM_B200_F32;
  using h16 = __half;
  using b16 = __nv_bfloat16;
  if (x == B && res == kNone) return pick_steps<b16, NoT>(k, drop);
  if (x == H && res == kNone) return pick_steps<h16, NoT>(k, drop);
  if (x == F && res == kNone) return pick_steps<float, NoT>(k, drop);
  if (x == B && res == B) return pick_steps<b16, b16>(k, drop);
  if (x == H && res == H) return pick_steps<h16, h16>(k, drop);
  if (x == F && res == F) return pick_steps<float, float>(k, drop);
  if (x == B && res == F) return pick_steps<b16, float>(k, drop);
  if (x == H && res == F) return pick_steps<h16, float>(k, drop);
  return nullptr;
}

int launch_generic(const FusedFwdParams& p, bool drop, UnitDevice* ud, cudaStream_t stream, const char* why) {
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(p.rows, int64_t{8} * ud->sm_count));
  if (drop)
    fused_fwd_generic_kernel<true><<<grid, kGenericThreads, 0, stream>>>(p);
  else
    fused_fwd_generic_kernel<false><<<grid, kGenericThreads, 0, stream>>>(p);
  return launched(std::string("fused_fwd_generic (") + why + ") grid=" + std::to_string(grid));
}

int run(const FusedFwdParams& p, bool drop, cudaStream_t stream) {
  UnitDevice* ud = nullptr;
  int st = unit_device(&ud);
  if (st) return st;
  Ranges ranges;
  const size_t n = static_cast<size_t>(p.rows) * static_cast<size_t>(p.N);
  ranges.add(p.x, n * elem_bytes(p.x_dt));
  if (p.res) ranges.add(p.res, n * elem_bytes(p.res_dt));
  if (p.w) ranges.add(p.w, p.N * elem_bytes(p.w_dt));
  if (p.b) ranges.add(p.b, p.N * elem_bytes(p.b_dt));
  ranges.add(p.out, n * (p.scales ? 1 : elem_bytes(p.out_dt)));
  if (p.ro) ranges.add(p.ro, n * elem_bytes(p.ro_dt));
  if (p.rstd) ranges.add(p.rstd, p.rows * 4);
  if (p.scales) {
    const int64_t groups = p.group ? (p.N + p.group - 1) / p.group : 1;
    ranges.add(p.scales, ((p.rows - 1) * p.scale_row + (groups - 1) * p.scale_group + 1) * 4);
  }
  if (p.drop.step) ranges.add(p.drop.step, 8);
  st = ranges.send(stream);
  if (st) return st;
  const void* ptrs[] = {p.x, p.res, p.out, p.ro};
  const char* why = p.N % 8 ? "hidden % 8" : nullptr;
  for (const void* ptr : ptrs)
    if (!aligned_to(ptr, ptr == p.out && p.scales ? 8 : 16)) why = "unaligned pointer";
  if (!why) {
    const int bytes[3] = {elem_bytes(p.x_dt), p.res ? elem_bytes(p.res_dt) : 0, 0};
    RowPlan pl;
    int k = 0, smem = 0;
    why = plan_rows(p.rows, p.N, bytes, p.b != nullptr, kRowMaxVecs, ud->sm_count, &pl, &k, &smem);
    if (!why) {
      FwdKernel kernel = pick(p.x_dt, p.res ? p.res_dt : kNone, k, drop);
      if (kernel) {
        st = launch_rows(ud, kernel, p, pl, smem, stream, drop ? "dropout_fwd" : "quant_fwd", k);
        if (st != RMSNORM_B200_ERR_UNSUPPORTED) return st;
        why = "cluster not schedulable";
      } else {
        why = "dtype combination";
      }
    }
  }
  return launch_generic(p, drop, ud, stream, why);
}

}  // namespace
}  // namespace rmsb200

using namespace rmsb200;

extern "C" int rmsnorm_b200_quant_fwd(const rmsnorm_b200_quant_args* a, void* stream) {
  if (!a || a->rows < 0 || a->hidden < 1) return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (!valid_dt(a->x_dtype) || (a->q_dtype != RMSNORM_B200_E4M3 && a->q_dtype != RMSNORM_B200_I8))
    return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if ((a->residual && !valid_dt(a->residual_dtype)) || (a->residual_out && !valid_dt(a->residual_out_dtype)) ||
      (a->weight && !valid_dt(a->weight_dtype)) || (a->bias && !valid_dt(a->bias_dtype)))
    return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (a->group != 0 && a->group != 32 && a->group != 64 && a->group != 128 && a->group != 256)
    return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (a->scale_row_stride < 0 || a->scale_group_stride < 0) return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (a->rows > 0 && (!a->x || !a->q || !a->scales)) return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (a->rows == 0) {
    rmsb_units::set_last_plan("quant empty");
    return RMSNORM_B200_OK;
  }
  FusedFwdParams p = {};
  p.x = a->x; p.res = a->residual; p.w = a->weight; p.b = a->bias;
  p.out = a->q; p.ro = a->residual_out; p.scales = a->scales;
  p.rows = a->rows; p.N = a->hidden;
  p.scale_row = a->scale_row_stride; p.scale_group = a->scale_group_stride;
  p.x_dt = a->x_dtype; p.res_dt = a->residual_dtype; p.w_dt = a->weight_dtype; p.b_dt = a->bias_dtype;
  p.out_dt = a->q_dtype; p.ro_dt = a->residual_out_dtype;
  p.group = a->group; p.eps = a->eps;
  return run(p, false, static_cast<cudaStream_t>(stream));
}

extern "C" int rmsnorm_b200_dropout_rmsnorm_fwd(const rmsnorm_b200_dropout_fwd_args* a, void* stream) {
  if (!a || a->rows < 0 || a->hidden < 1) return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (!valid_dt(a->x_dtype) || !valid_dt(a->out_dtype)) return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if ((a->residual && !valid_dt(a->residual_dtype)) || (a->residual_out && !valid_dt(a->residual_out_dtype)) ||
      (a->weight && !valid_dt(a->weight_dtype)) || (a->bias && !valid_dt(a->bias_dtype)))
    return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (!valid_drop(a->drop, a->rows)) return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (a->rows > 0 && (!a->x || !a->out)) return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (a->rows == 0) {
    rmsb_units::set_last_plan("dropout fwd empty");
    return RMSNORM_B200_OK;
  }
  FusedFwdParams p = {};
  p.x = a->x; p.res = a->residual; p.w = a->weight; p.b = a->bias;
  p.out = a->out; p.ro = a->residual_out; p.rstd = a->rstd;
  p.rows = a->rows; p.N = a->hidden;
  p.x_dt = a->x_dtype; p.res_dt = a->residual_dtype; p.w_dt = a->weight_dtype; p.b_dt = a->bias_dtype;
  p.out_dt = a->out_dtype; p.ro_dt = a->residual_out_dtype;
  p.eps = a->eps;
  expand_drop(a->drop, &p.drop);
  return run(p, true, static_cast<cudaStream_t>(stream));
}
