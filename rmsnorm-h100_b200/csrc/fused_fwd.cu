// fused_fwd.cu -- rmsnorm_b200_quant_fwd and rmsnorm_b200_dropout_rmsnorm_fwd: argument
// checks, plan and launch.
#define RMSB_UNIT fused_fwd
#include "unit_state.cuh"

#include "fused_fwd_kernels.cuh"
#include "odd_kernels.cuh"
#include "row_plan.h"
#include "shift_fwd_kernel.cuh"

namespace rmsb200 {
namespace {

using FwdKernel = void (*)(const FusedFwdParams, const RowPlan);
constexpr int kNone = -1;

// What a row ends as: dropout, or an 8-bit type with one scale per row or per group.
enum End { kDropped, kE4M3Row, kE4M3Group, kI8Row, kI8Group };

template <typename X, typename RT, typename ROT, typename E>
FwdKernel pick_steps(int k) {
  switch (k) {
    case 1: return fused_fwd_kernel<X, RT, ROT, E, 1>;
    case 2: return fused_fwd_kernel<X, RT, ROT, E, 2>;
    default: return fused_fwd_kernel<X, RT, ROT, E, 4>;
  }
}

template <typename X, typename RT, typename ROT>
FwdKernel pick_quant(int end, int k) {
  switch (end) {
    case kE4M3Row: return pick_steps<X, RT, ROT, Scaled<E4M3, true>>(k);
    case kE4M3Group: return pick_steps<X, RT, ROT, Scaled<E4M3, false>>(k);
    case kI8Row: return pick_steps<X, RT, ROT, Scaled<I8, true>>(k);
    case kI8Group: return pick_steps<X, RT, ROT, Scaled<I8, false>>(k);
    default: return nullptr;
  }
}

// Types of x, residual and residual_out: the residual stream in x's type, in fp32, or turned
// from x's type into fp32. The output of dropout has x's type.
FwdKernel pick(int x, int res, int ro, int end, int k) {
  constexpr int H = RMSNORM_B200_F16, B = RMSNORM_B200_BF16, F = RMSNORM_B200_F32;
  using h16 = __half;
  using b16 = __nv_bfloat16;
#define RMSB_FUSED(XC, RC, ROC, X, RT, ROT)  \
  if (x == XC && res == RC && ro == ROC)     \
    return end == kDropped ? pick_steps<X, RT, ROT, Dropped>(k) : pick_quant<X, RT, ROT>(end, k);
#define RMSB_QUANT(XC, X) \
  if (x == XC && res == kNone && ro == kNone) return pick_quant<X, NoT, NoT>(end, k);
#define RMSB_DROP(XC, ROC, X, ROT) \
  if (x == XC && res == kNone && ro == ROC && end == kDropped) return pick_steps<X, NoT, ROT, Dropped>(k);
  RMSB_FUSED(B, B, B, b16, b16, b16)
  RMSB_FUSED(H, H, H, h16, h16, h16)
  RMSB_FUSED(F, F, F, float, float, float)
  RMSB_FUSED(B, B, F, b16, b16, float)
  RMSB_FUSED(H, H, F, h16, h16, float)
  RMSB_FUSED(B, F, F, b16, float, float)
  RMSB_FUSED(H, F, F, h16, float, float)
  RMSB_QUANT(B, b16)
  RMSB_QUANT(H, h16)
  RMSB_QUANT(F, float)
  RMSB_DROP(B, B, b16, b16)
  RMSB_DROP(H, H, h16, h16)
  RMSB_DROP(F, F, float, float)
  RMSB_DROP(B, F, b16, float)
  RMSB_DROP(H, F, h16, float)
#undef RMSB_FUSED
#undef RMSB_QUANT
#undef RMSB_DROP
  return nullptr;
}

template <typename X, typename RO>
FwdKernel pick_odd(bool drop, int k) {
  if (drop) return k == 1 ? odd_fwd_kernel<X, RO, false, 1> : k == 2 ? odd_fwd_kernel<X, RO, false, 2> : odd_fwd_kernel<X, RO, false, 4>;
  return k == 1 ? odd_fwd_kernel<X, RO, true, 1> : k == 2 ? odd_fwd_kernel<X, RO, true, 2> : odd_fwd_kernel<X, RO, true, 4>;
}

FwdKernel pick_odd(const FusedFwdParams& p, bool drop, int k) {
  constexpr int H = RMSNORM_B200_F16, B = RMSNORM_B200_BF16, F = RMSNORM_B200_F32;
  const int x = p.x_dt, ro = p.ro ? p.ro_dt : x;
  if ((p.res && p.res_dt != x) || (drop && p.out_dt != x)) return pick_odd<Any, Any>(drop, k);
  if (x == B && ro == B) return pick_odd<__nv_bfloat16, __nv_bfloat16>(drop, k);
  if (x == H && ro == H) return pick_odd<__half, __half>(drop, k);
  if (x == F && ro == F) return pick_odd<float, float>(drop, k);
  if (x == B && ro == F) return pick_odd<__nv_bfloat16, float>(drop, k);
  if (x == H && ro == F) return pick_odd<__half, float>(drop, k);
  return pick_odd<Any, Any>(drop, k);
}

template <typename X, typename E>
FwdKernel pick_shift(int k) {
  return k == 1 ? shift_fwd_kernel<X, E, 1> : shift_fwd_kernel<X, E, kShiftFwdSteps>;
}

template <typename X>
FwdKernel pick_shift(int end, int k) {
  switch (end) {
    case kDropped: return pick_shift<X, Dropped>(k);
    case kE4M3Row: return pick_shift<X, Scaled<E4M3, true>>(k);
    case kE4M3Group: return pick_shift<X, Scaled<E4M3, false>>(k);
    case kI8Row: return pick_shift<X, Scaled<I8, true>>(k);
    case kI8Group: return pick_shift<X, Scaled<I8, false>>(k);
    default: return nullptr;
  }
}

FwdKernel pick_shift(int x, int end, int k) {
  if (x == RMSNORM_B200_F32) return pick_shift<float>(end, k);
  return x == RMSNORM_B200_BF16 ? pick_shift<__nv_bfloat16>(end, k) : pick_shift<__half>(end, k);
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
  ranges.add_out(p.out, n * (p.scales ? 1 : elem_bytes(p.out_dt)));
  if (p.ro) ranges.add(p.ro, n * elem_bytes(p.ro_dt));
  if (p.rstd) ranges.add(p.rstd, p.rows * 4);
  if (p.scales) {
    const int64_t groups = p.group ? (p.N + p.group - 1) / p.group : 1;
    ranges.add(p.scales, ((p.rows - 1) * p.scale_row + (groups - 1) * p.scale_group + 1) * 4);
  }
  if (p.drop.step) ranges.add(p.drop.step, 8);
  st = ranges.send(stream);
  if (st) return st;
  // Aligned tensors in a combination of types with a kernel of its own: whole vectors where rows
  // consist of them, shifted ones where they do not; else the odd rows' kernels; else (rows wider
  // than a cluster holds) the generic one.
  const int bytes[3] = {elem_bytes(p.x_dt), p.res ? elem_bytes(p.res_dt) : 0, 0};
  RowPlan pl;
  int k = 0, smem = 0;
  const void* ptrs[] = {p.x, p.res, p.out, p.ro};
  bool aligned = !drop || p.out_dt == p.x_dt;
  for (const void* ptr : ptrs) aligned = aligned && aligned_to(ptr, ptr == p.out && p.scales ? 8 : 16);
  const bool i8 = p.out_dt == RMSNORM_B200_I8;
  const int end = drop ? kDropped : p.group ? (i8 ? kI8Group : kE4M3Group) : (i8 ? kI8Row : kE4M3Row);
  const char* why = nullptr;
  if (aligned && p.N % 8 == 0) {
    const bool few = p.rows <= ud->sm_count && p.N <= kFwdFewThreads * 8;
    why = plan_rows(p.rows, p.N, bytes, p.b != nullptr, few ? kFwdFewThreads : kFwdThreads, few ? 1 : kFwdSteps,
                    ud->sm_count, &pl, &k, &smem);
    if (!why) {
      if (FwdKernel kernel = pick(p.x_dt, p.res ? p.res_dt : kNone, p.ro ? p.ro_dt : kNone, end, k)) {
        st = launch_rows(ud, kernel, p, pl, smem, stream, drop ? "dropout_fwd" : "quant_fwd", k);
        if (st != RMSNORM_B200_ERR_UNSUPPORTED) return st;
      }
    }
  } else if (aligned && (!p.res || p.res_dt == p.x_dt || p.res_dt == RMSNORM_B200_F32) &&
             (!p.ro || p.ro_dt == p.x_dt || p.ro_dt == RMSNORM_B200_F32)) {
    RowWants want;
    want.shifted = true;
    want.scale = p.group;
    why = plan_rows(p.rows, shifted_columns(p.N), bytes, p.b != nullptr, kShiftThreads, kShiftFwdSteps, ud->sm_count,
                    &pl, &k, &smem, want);
    if (!why && !(p.group && pl.C > 1)) {  // a scale's columns may lie in two CTAs' slices
      FwdKernel kernel = pick_shift(p.x_dt, end, k);
      st = launch_shifted(ud, kernel, p, pl, smem, stream, drop ? "dropout_fwd_sh" : "quant_fwd_sh", k);
      if (st != RMSNORM_B200_ERR_UNSUPPORTED) return st;
    }
  }
  RowWants want;
  want.odd = true;
  why = plan_rows(p.rows, p.N, bytes, p.b != nullptr, kOddThreads, kOddSteps, ud->sm_count, &pl, &k, &smem, want);
  if (!why) {
    st = launch_rows(ud, pick_odd(p, drop, k), p, pl, smem, stream,
                     drop ? "dropout_fwd_odd" : "quant_fwd_odd", k);
    if (st != RMSNORM_B200_ERR_UNSUPPORTED) return st;
    why = "cluster not schedulable";
  }
  return launch_generic(p, drop, ud, stream, why);
}

int quant_fwd(const rmsnorm_b200_quant_args* a, void* stream) {
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
  while (p.group >> p.group_shift > 1) ++p.group_shift;
  return run(p, false, static_cast<cudaStream_t>(stream));
}

int dropout_fwd(const rmsnorm_b200_dropout_fwd_args* a, void* stream) {
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

}  // namespace
}  // namespace rmsb200

using namespace rmsb200;

extern "C" int rmsnorm_b200_quant_fwd(const rmsnorm_b200_quant_args* a, void* stream) {
  return entry([&] { return quant_fwd(a, stream); });
}

extern "C" int rmsnorm_b200_dropout_rmsnorm_fwd(const rmsnorm_b200_dropout_fwd_args* a, void* stream) {
  return entry([&] { return dropout_fwd(a, stream); });
}
