// fused_fwd.cu -- rmsnorm_b200_quant_fwd and rmsnorm_b200_dropout_rmsnorm_fwd: argument
// checks, plan and launch.
#define RMSB_UNIT fused_fwd
#include "unit_state.cuh"

#include "fused_generic.cuh"

namespace rmsb200 {
namespace {

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
  return launch_generic(p, drop, ud, stream, "plain");
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
