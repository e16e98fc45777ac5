// fused_bwd.cu -- rmsnorm_b200_dropout_rmsnorm_bwd: argument checks, plan and launch.
#define RMSB_UNIT fused_bwd
#include "unit_state.cuh"

#include "column_sums.cuh"
#include "fused_bwd_kernels.cuh"
#include "odd_kernels.cuh"
#include "row_plan.h"
#include "shift_bwd_kernel.cuh"

namespace rmsb200 {
namespace {

using BwdKernel = void (*)(const FusedBwdParams, const RowPlan);

struct Plan {
  int64_t nparts = 0;      // partial rows of dweight / dbias
  int64_t chunk_rows = 1;  // generic path: rows per partial row
  BwdKernel kernel = nullptr;
  RowPlan rows;
  int k = 0, smem = 0;
  const char* kind = "";
  const char* why = nullptr;  // why the generic path is taken
};

// g: threads of a row group where the kernel has them built in, else 0.
template <typename H, typename DY, typename DRO, typename DRES>
BwdKernel pick_steps(int k, int g) {
  // four steps hold a row of 16-bit values only
  if constexpr (sizeof(H) == 2 && sizeof(DY) == 2) {
    switch (g) {
      case 32: return fused_bwd_kernel<H, DY, DRO, DRES, kBwdTmemSteps, 32>;
      case 64: return fused_bwd_kernel<H, DY, DRO, DRES, kBwdTmemSteps, 64>;
      case 96: return fused_bwd_kernel<H, DY, DRO, DRES, kBwdTmemSteps, 96>;
      case 128: return fused_bwd_kernel<H, DY, DRO, DRES, kBwdTmemSteps, 128>;
      case 160: return fused_bwd_kernel<H, DY, DRO, DRES, kBwdTmemSteps, 160>;
      case 192: return fused_bwd_kernel<H, DY, DRO, DRES, kBwdTmemSteps, 192>;
      case 256: return fused_bwd_kernel<H, DY, DRO, DRES, kBwdTmemSteps, 256>;
      case 320: return fused_bwd_kernel<H, DY, DRO, DRES, kBwdTmemSteps, 320>;
      case 384: return fused_bwd_kernel<H, DY, DRO, DRES, kBwdTmemSteps, 384>;
      case 512: return fused_bwd_kernel<H, DY, DRO, DRES, kBwdTmemSteps, 512>;
    }
  }
  return k == 1 ? fused_bwd_kernel<H, DY, DRO, DRES, 1, 0> : fused_bwd_kernel<H, DY, DRO, DRES, 2, 0>;
}

// The smallest of them that holds a row's `threads`, or the largest.
int built_in_group(int64_t threads) {
  for (const int g : {32, 64, 96, 128, 160, 192, 256, 320, 384})
    if (threads <= g) return g;
  return kBwdThreads;
}

template <typename H, typename DY>
BwdKernel pick_residual(bool dro, bool dres, int k, int g) {
  if (dro) return dres ? pick_steps<H, DY, H, H>(k, g) : pick_steps<H, DY, H, NoT>(k, g);
  return dres ? pick_steps<H, DY, NoT, H>(k, g) : pick_steps<H, DY, NoT, NoT>(k, g);
}

// The saved input in dout's type or in fp32; dresidual_out and dresidual have its type, dx has
// dout's.
BwdKernel pick(const rmsnorm_b200_dropout_bwd_args* a, int k, int g) {
  constexpr int H = RMSNORM_B200_F16, B = RMSNORM_B200_BF16, F = RMSNORM_B200_F32;
  using h16 = __half;
  using b16 = __nv_bfloat16;
  const int h = a->h_dtype, dy = a->dout_dtype;
  const bool dro = a->dresidual_out, dres = a->dresidual;
  if (a->dx_dtype != dy || (dro && a->dresidual_out_dtype != h) || (dres && a->dresidual_dtype != h)) return nullptr;
  if (h == B && dy == B) return pick_residual<b16, b16>(dro, dres, k, g);
  if (h == H && dy == H) return pick_residual<h16, h16>(dro, dres, k, g);
  if (h == F && dy == F) return pick_residual<float, float>(dro, dres, k, g);
  if (h == F && dy == B) return pick_residual<float, b16>(dro, dres, k, g);
  if (h == F && dy == H) return pick_residual<float, h16>(dro, dres, k, g);
  return nullptr;
}

template <typename H, typename DY>
BwdKernel pick_odd(int k) {
  return k == 1 ? odd_bwd_kernel<H, DY, 1> : odd_bwd_kernel<H, DY, 2>;
}

BwdKernel pick_odd(const rmsnorm_b200_dropout_bwd_args* a, int k) {
  constexpr int H = RMSNORM_B200_F16, B = RMSNORM_B200_BF16, F = RMSNORM_B200_F32;
  const int h = a->h_dtype, dy = a->dout_dtype;
  if (a->dx_dtype != dy || (a->dresidual_out && a->dresidual_out_dtype != h) ||
      (a->dresidual && a->dresidual_dtype != h))
    return pick_odd<Any, Any>(k);
  if (h == B && dy == B) return pick_odd<__nv_bfloat16, __nv_bfloat16>(k);
  if (h == H && dy == H) return pick_odd<__half, __half>(k);
  if (h == F && dy == F) return pick_odd<float, float>(k);
  if (h == F && dy == B) return pick_odd<float, __nv_bfloat16>(k);
  if (h == F && dy == H) return pick_odd<float, __half>(k);
  return pick_odd<Any, Any>(k);
}

int check(const rmsnorm_b200_dropout_bwd_args* a) {
  if (!a || a->rows < 0 || a->hidden < 1) return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (!valid_dt(a->h_dtype) || !valid_dt(a->dout_dtype) || !valid_dt(a->dx_dtype))
    return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if ((a->weight && !valid_dt(a->weight_dtype)) || (a->dresidual_out && !valid_dt(a->dresidual_out_dtype)) ||
      (a->dresidual && !valid_dt(a->dresidual_dtype)) || (a->dweight && !valid_dt(a->dweight_dtype)) ||
      (a->dbias && !valid_dt(a->dbias_dtype)))
    return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (!valid_drop(a->drop, a->rows)) return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (a->rows > 0 && (!a->h || !a->dout || !a->rstd || !a->dx)) return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  return RMSNORM_B200_OK;
}

BwdKernel pick_shift(const rmsnorm_b200_dropout_bwd_args* a) {
  constexpr int H = RMSNORM_B200_F16, B = RMSNORM_B200_BF16, F = RMSNORM_B200_F32;
  const int h = a->h_dtype, dy = a->dout_dtype;
  if (a->dx_dtype != dy || (a->dresidual_out && a->dresidual_out_dtype != h) ||
      (a->dresidual && a->dresidual_dtype != h))
    return nullptr;
  if (h == B && dy == B) return shift_bwd_kernel<__nv_bfloat16, __nv_bfloat16>;
  if (h == H && dy == H) return shift_bwd_kernel<__half, __half>;
  if (h == F && dy == F) return shift_bwd_kernel<float, float>;
  if (h == F && dy == B) return shift_bwd_kernel<float, __nv_bfloat16>;
  if (h == F && dy == H) return shift_bwd_kernel<float, __half>;
  return nullptr;
}

int make_plan(UnitDevice* ud, const rmsnorm_b200_dropout_bwd_args* a, Plan* pl) {
  // Aligned tensors in a combination of types with a kernel of its own: whole vectors where rows
  // consist of them, shifted ones where they do not; else the odd rows' kernels; else (rows
  // wider than a cluster holds) the generic ones.
  const int bytes[3] = {elem_bytes(a->h_dtype), elem_bytes(a->dout_dtype),
                        a->dresidual_out ? elem_bytes(a->dresidual_out_dtype) : 0};
  const void* ptrs[] = {a->h, a->dout, a->dresidual_out, a->dx, a->dresidual};
  bool aligned = true;
  for (const void* ptr : ptrs) aligned = aligned && aligned_to(ptr, 16);
  for (const bool odd : {false, true}) {
    if (!odd && !aligned) continue;
    bool shifted = !odd && a->hidden % 8 != 0;
    RowWants want;
    if (odd) {
      want.odd = true;
      pl->why = plan_rows(a->rows, a->hidden, bytes, false, kOddThreads, kOddBwdSteps, ud->sm_count, &pl->rows, &pl->k,
                          &pl->smem, want);
      pl->kernel = pick_odd(a, pl->k);
    } else if (!shifted) {
      // 16-bit rows that fill more than two steps of a warp: four steps a thread, sums in tensor
      // memory, by groups of the size that fits (32263 x 4160: three of 160 threads 279 us, two of
      // 256 365 us). The others, and few rows (a CTA each, as many threads as it has): registers.
      const bool few = a->rows <= ud->sm_count && a->hidden <= kBwdThreads * 8 * kBwdRegSteps;
      if (!few && a->h_dtype != RMSNORM_B200_F32 && a->dout_dtype == a->h_dtype && a->hidden > 32 * 8 * kBwdRegSteps)
        want.built_in = built_in_group((a->hidden + 8 * kBwdTmemSteps - 1) / (8 * kBwdTmemSteps));
      pl->why = plan_rows(a->rows, a->hidden, bytes, false, kBwdThreads, want.built_in ? kBwdTmemSteps : kBwdRegSteps,
                          ud->sm_count, &pl->rows, &pl->k, &pl->smem, want);
      if (want.built_in) pl->k = kBwdTmemSteps;
      pl->kernel = pl->why ? nullptr : pick(a, pl->k, want.built_in);
      // A CTA's single row of which two steps in registers leave a third of the threads idle goes to
      // the shifted kernel, which holds four steps: 32263 x 4160, fp32 h, bf16 dout 406 against 564 us.
      if (!pl->why && !few && !want.built_in && pl->k == kBwdRegSteps && pl->rows.groups == 1 &&
          pl->rows.slice * 3 < kBwdThreads * kBwdRegSteps * 8 * 2)
        shifted = true;
    }
    if (shifted) {
      // four steps a thread where two whole rows fit the ring, or 16-bit rows one at least; wider
      // ones are split
      const int elem = bytes[0] + bytes[1] + bytes[2];
      const bool two_fit = 2 * shifted_columns(a->hidden) * elem <= kRingBytes;
      const int steps = two_fit || elem <= 6 ? kShiftBwdSteps : kShiftBwdSteps / 2;
      want.shifted = want.whole = true;
      pl->why = plan_rows(a->rows, shifted_columns(a->hidden), bytes, false, kShiftThreads, steps, ud->sm_count,
                          &pl->rows, &pl->k, &pl->smem, want);
      pl->kernel = pick_shift(a);
    }
    if (pl->why) pl->kernel = nullptr;
    if (!pl->kernel) continue;
    pl->kind = odd ? "dropout_bwd_odd" : shifted ? "dropout_bwd_sh" : "dropout_bwd";
    // the groups' sums of a vector step pass through the rings
    if (odd || shifted || pl->rows.groups > 1) pl->smem = std::max(pl->smem, kBwdThreads * 64);
    int grid = 0;
    const int st = (shifted ? launch_shifted<BwdKernel, FusedBwdParams> : launch_rows<BwdKernel, FusedBwdParams>)(
        ud, pl->kernel, FusedBwdParams{}, pl->rows, pl->smem, nullptr, "", pl->k, &grid, true);
    if (st == RMSNORM_B200_OK) {
      pl->nparts = a->dweight || a->dbias ? grid / pl->rows.C : 0;
      return st;
    }
    if (st != RMSNORM_B200_ERR_UNSUPPORTED) return st;
    pl->kernel = nullptr;
    pl->why = "cluster not schedulable";
  }
  if (!a->dweight && !a->dbias) return RMSNORM_B200_OK;
  const int64_t col_blocks = (a->hidden + kGenericThreads - 1) / kGenericThreads;
  const int64_t target = std::clamp<int64_t>((4 * ud->sm_count + col_blocks - 1) / col_blocks, 1, 1024);
  // at most 256 rows are added one after the other (longer runs lose digits of the sum), and
  // at most 65535 chunks fit a grid
  pl->chunk_rows = std::clamp<int64_t>((a->rows + target - 1) / target, 1, 256);
  pl->chunk_rows = std::max<int64_t>(pl->chunk_rows, (a->rows + 65534) / 65535);
  pl->nparts = (a->rows + pl->chunk_rows - 1) / pl->chunk_rows;
  return RMSNORM_B200_OK;
}

size_t workspace(const rmsnorm_b200_dropout_bwd_args* a, const Plan& pl) {
  const size_t per = static_cast<size_t>(pl.nparts) * static_cast<size_t>(a->hidden) * sizeof(float);
  return (a->dweight ? per : 0) + (a->dbias ? per : 0);
}

int launch_generic(const FusedBwdParams& p, const Plan& pl, UnitDevice* ud, cudaStream_t stream, const char* why) {
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(p.rows, int64_t{8} * ud->sm_count));
  fused_bwd_generic_kernel<<<grid, kGenericThreads, 0, stream>>>(p);
  int st = launched(std::string("fused_bwd_generic (") + why + ") grid=" + std::to_string(grid) +
                    " chunks=" + std::to_string(pl.nparts));
  if (st || (!p.dw_part && !p.db_part)) return st;
  GenBwdParams g = {};
  g.rows = p.rows; g.N = p.N; g.H = 1;
  g.x = p.h; g.x_dt = p.h_dt; g.dy = p.dy; g.dy_dt = p.dy_dt; g.rstd = p.rstd;
  const dim3 pg(static_cast<unsigned>((p.N + kGenericThreads - 1) / kGenericThreads),
                static_cast<unsigned>(pl.nparts));
  bwd_generic_partials_kernel<<<pg, kGenericThreads, 0, stream>>>(g, pl.chunk_rows, p.dw_part, p.db_part);
  return launched("");
}

int run(const rmsnorm_b200_dropout_bwd_args* a, void* ws, size_t ws_bytes, cudaStream_t stream) {
  int st = check(a);
  if (st) return st;
  UnitDevice* ud = nullptr;
  st = unit_device(&ud);
  if (st) return st;
  Plan pl;
  st = make_plan(ud, a, &pl);
  if (st) return st;
  const size_t need = workspace(a, pl);
  if (need > ws_bytes || (need > 0 && (!ws || !aligned_to(ws, 16)))) return RMSNORM_B200_ERR_WORKSPACE;
  Ranges ranges;
  const size_t n = static_cast<size_t>(a->rows) * static_cast<size_t>(a->hidden);
  ranges.add(a->h, n * elem_bytes(a->h_dtype));
  ranges.add(a->dout, n * elem_bytes(a->dout_dtype));
  ranges.add(a->rstd, static_cast<size_t>(a->rows) * 4);
  if (a->weight) ranges.add(a->weight, a->hidden * elem_bytes(a->weight_dtype));
  if (a->dresidual_out) ranges.add(a->dresidual_out, n * elem_bytes(a->dresidual_out_dtype));
  ranges.add(a->dx, n * elem_bytes(a->dx_dtype));
  if (a->dresidual) ranges.add(a->dresidual, n * elem_bytes(a->dresidual_dtype));
  if (a->dweight) ranges.add(a->dweight, a->hidden * elem_bytes(a->dweight_dtype));
  if (a->dbias) ranges.add(a->dbias, a->hidden * elem_bytes(a->dbias_dtype));
  if (a->drop.step) ranges.add(a->drop.step, 8);
  ranges.add(ws, need);
  st = ranges.send(stream);
  if (st) return st;

  FusedBwdParams p = {};
  p.h = a->h; p.dy = a->dout; p.rstd = a->rstd; p.w = a->weight; p.dro = a->dresidual_out;
  p.dx = a->dx; p.dres = a->dresidual;
  p.rows = a->rows; p.N = a->hidden;
  p.h_dt = a->h_dtype; p.dy_dt = a->dout_dtype; p.w_dt = a->weight_dtype; p.dro_dt = a->dresidual_out_dtype;
  p.dx_dt = a->dx_dtype; p.dres_dt = a->dresidual_dtype;
  p.dw_part = a->dweight ? static_cast<float*>(ws) : nullptr;
  p.db_part = a->dbias ? static_cast<float*>(ws) + (a->dweight ? pl.nparts * a->hidden : 0) : nullptr;
  expand_drop(a->drop, &p.drop);
  if (a->rows > 0) {
    st = pl.kernel ? launch_rows(ud, pl.kernel, p, pl.rows, pl.smem, stream, pl.kind, pl.k)
                   : launch_generic(p, pl, ud, stream, pl.why);
    if (st) return st;
  } else {
    rmsb_units::set_last_plan("dropout bwd empty");
  }
  // dweight and dbias: fixed-order column sums of the partial rows, one launch for both
  ReduceParams rp = {};
  rp.C = a->rows > 0 ? pl.nparts : 0;
  rp.W = a->hidden;
  rp.N = a->hidden;
  int njobs = 0;
  int64_t blocks = 0;
  auto add_job = [&](const float* part, void* out, int dt) {
    ReduceJob& jb = rp.job[njobs++];
    jb.part = part;
    jb.out = out;
    jb.wout = a->hidden;
    jb.fold = 1;
    jb.out_dt = dt;
    const int64_t cols = reduce_vectorised(jb, rp.W) ? kReduceVCols : kReduceCols;
    blocks = std::max(blocks, (jb.wout + cols - 1) / cols);
  };
  if (a->dweight) add_job(p.dw_part, a->dweight, a->dweight_dtype);
  if (a->dbias) add_job(p.db_part, a->dbias, a->dbias_dtype);
  if (njobs == 0) return RMSNORM_B200_OK;
  reduce_partials_kernel<<<dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(njobs)), kReduceThreads, 0,
                           stream>>>(rp);
  return launched("");
}

int workspace_size(const rmsnorm_b200_dropout_bwd_args* a, size_t* bytes) {
  if (!bytes) return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  *bytes = 0;
  int st = check(a);
  if (st) return st;
  UnitDevice* ud = nullptr;
  st = unit_device(&ud);
  if (st) return st;
  Plan pl;
  st = make_plan(ud, a, &pl);
  if (st) return st;
  *bytes = workspace(a, pl);
  return RMSNORM_B200_OK;
}

}  // namespace
}  // namespace rmsb200

using namespace rmsb200;

extern "C" int rmsnorm_b200_dropout_rmsnorm_bwd_workspace_size(const rmsnorm_b200_dropout_bwd_args* a,
                                                               size_t* bytes) {
  return entry([&] { return workspace_size(a, bytes); });
}

extern "C" int rmsnorm_b200_dropout_rmsnorm_bwd(const rmsnorm_b200_dropout_bwd_args* a, void* workspace,
                                                size_t workspace_bytes, void* stream) {
  return entry([&] { return run(a, workspace, workspace_bytes, static_cast<cudaStream_t>(stream)); });
}
