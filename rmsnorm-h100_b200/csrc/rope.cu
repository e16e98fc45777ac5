// rope.cu -- rmsnorm_b200_rope_fwd and rmsnorm_b200_rope_bwd: argument checks, plan and launch.
#define RMSB_UNIT rope
#include "unit_state.cuh"

#include <cstring>

#include "column_sums.cuh"
#include "rope_kernels.cuh"

namespace rmsb200 {
namespace {

bool valid_tensor(const rmsnorm_b200_rope_tensor& t, int64_t tokens, int heads) {
  return heads == 0 || tokens == 0 || (t.data && t.token_stride >= 0 && t.head_stride >= 0);
}

int check(const rmsnorm_b200_rope_args* a) {
  if (!a || a->tokens < 0 || a->q_heads < 1 || a->k_heads < 0) return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (a->q_heads > RMSNORM_B200_ROPE_MAX_HEADS || a->k_heads > RMSNORM_B200_ROPE_MAX_HEADS)
    return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (a->head_dim < 1 || a->head_dim > kRopeMaxDim || a->rotary_dim < 0 || a->rotary_dim > a->head_dim ||
      (a->rotary_dim & 1))
    return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (a->axes < 1 || a->axes > 4 || !valid_dt(a->dtype)) return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  for (int i = 0; i < a->rotary_dim / 2; ++i)
    if (static_cast<int>(a->axis_of_pair[i >> 5] >> (2 * (i & 31)) & 3) >= a->axes)
      return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if ((a->q_weight || a->k_weight) && !valid_dt(a->weight_dtype)) return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (a->q_weight && a->q_weight_heads != 1 && a->q_weight_heads != a->q_heads)
    return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (a->k_weight && a->k_weight_heads != 1 && a->k_weight_heads != a->k_heads)
    return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (!valid_tensor(a->q, a->tokens, a->q_heads) || !valid_tensor(a->k, a->tokens, a->k_heads))
    return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (a->tokens > 0 && a->rotary_dim > 0 &&
      (!a->positions || !a->table || a->table_rows < 0 || a->position_axis_stride < 0))
    return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  return RMSNORM_B200_OK;
}

void add_tensor(Ranges& r, const rmsnorm_b200_rope_tensor& t, const rmsnorm_b200_rope_args* a, int heads) {
  if (heads == 0) return;
  r.add(t.data, ((a->tokens - 1) * t.token_stride + (heads - 1) * t.head_stride + a->head_dim) *
                    elem_bytes(a->dtype));
}

void add_ranges(Ranges& r, const rmsnorm_b200_rope_args* a) {
  add_tensor(r, a->q, a, a->q_heads);
  add_tensor(r, a->k, a, a->k_heads);
  const size_t wb = static_cast<size_t>(a->head_dim) * elem_bytes(a->weight_dtype);
  if (a->q_weight) r.add(a->q_weight, a->q_weight_heads * wb);
  if (a->k_weight) r.add(a->k_weight, a->k_weight_heads * wb);
  if (a->rotary_dim == 0) return;
  r.add(a->positions, ((a->axes - 1) * a->position_axis_stride + a->tokens) * (a->positions_64bit ? 8 : 4));
  r.add(a->table, static_cast<size_t>(a->table_rows) * a->rotary_dim * 4);
}

RopeTensor tensor(const rmsnorm_b200_rope_tensor& t) { return {t.data, t.token_stride, t.head_stride}; }

RopeParams params(const rmsnorm_b200_rope_args* a) {
  RopeParams p = {};
  p.tokens = a->tokens; p.table_rows = a->table_rows;
  p.pos = a->positions; p.pos_axis = a->position_axis_stride; p.table = a->table;
  p.w[0] = a->q_weight; p.w[1] = a->k_weight;
  p.x[0] = tensor(a->q); p.x[1] = tensor(a->k);
  for (int i = 0; i < 4; ++i) p.axis_of[i] = a->axis_of_pair[i];
  p.heads[0] = a->q_heads; p.heads[1] = a->k_heads;
  p.w_per_head[0] = a->q_weight && a->q_weight_heads > 1;
  p.w_per_head[1] = a->k_weight && a->k_weight_heads > 1;
  p.D = a->head_dim; p.rd = a->rotary_dim; p.axes = a->axes; p.interleaved = a->interleaved != 0;
  p.norm = a->norm != 0; p.pos64 = a->positions_64bit != 0; p.dt = a->dtype; p.w_dt = a->weight_dtype;
  p.eps = a->eps;
  return p;
}

// Whether the vectorised kernels take these tensors: nothing but whole 16-byte granules.
bool vectorised(const rmsnorm_b200_rope_args* a, std::initializer_list<const rmsnorm_b200_rope_tensor*> tensors) {
  if (a->head_dim % 8 || a->rotary_dim % 8 || !aligned_to(a->table, 16) || a->table_rows > INT32_MAX) return false;
  const int granule = 16 / elem_bytes(a->dtype);
  for (const auto* t : tensors)
    if (t && (!aligned_to(t->data, 16) || t->token_stride % granule || t->head_stride % granule)) return false;
  return true;
}

constexpr int kRopeSlots = 8;         // ring slots of a warp, at most
constexpr int kRopeSmem = 208 * 1024;  // beside the backward's 16 KB of static shared memory

// Whether a tensor's heads are not neighbours.
bool heads_apart(const rmsnorm_b200_rope_tensor& t, int heads, int head_dim) {
  return heads > 1 && t.head_stride != head_dim;
}

struct RopeGrid {
  RopePlan pl;
  dim3 grid;
  int threads, smem;
};

// u: heads a lane works on. tensors: that stream through a warp's ring (0: no ring); apart: some
// of them head by head, which a warp's 32 lanes copy one each.
RopeGrid plan(const rmsnorm_b200_rope_args* a, int u, int tensors, bool apart, int sms) {
  RopeGrid g = {};
  RopePlan& pl = g.pl;
  while ((8 << pl.lanes_shift) < a->head_dim) ++pl.lanes_shift;
  const int heads = pl.warp_heads = std::min(u * (32 >> pl.lanes_shift), apart ? 32 : INT32_MAX);
  pl.jobs[0] = (a->q_heads + heads - 1) / heads;
  pl.jobs[1] = (a->k_heads + heads - 1) / heads;
  pl.turned_lanes = a->rotary_dim / 8;
  const int jobs = pl.jobs[0] + pl.jobs[1];
  pl.cta_jobs = std::min(jobs, kRopeWarps);
  const int at_once = static_cast<int>(std::clamp<int64_t>(a->tokens, 1, kRopeWarps / pl.cta_jobs));
  const int warps = at_once * pl.cta_jobs;
  g.threads = warps * 32;
  const int64_t across = (jobs + pl.cta_jobs - 1) / pl.cta_jobs;
  // one CTA an SM where its rings take the shared memory
  const int64_t most = std::max<int64_t>(1, (tensors ? 1 : 2) * static_cast<int64_t>(sms) / across);
  const int64_t along = std::clamp<int64_t>((a->tokens + at_once - 1) / at_once, 1, most);
  g.grid = dim3(static_cast<unsigned>(along), static_cast<unsigned>(across));
  if (tensors) {
    pl.slot_bytes = static_cast<uint32_t>(heads * a->head_dim * elem_bytes(a->dtype));
    const int slot = warps * tensors * static_cast<int>(pl.slot_bytes) + warps * 8;
    const int64_t tokens = (a->tokens + along * at_once - 1) / (along * at_once);  // of a warp
    pl.S = static_cast<int>(std::clamp<int64_t>(tokens, 1, std::min(kRopeSlots, kRopeSmem / slot)));
    g.smem = pl.S * slot;
  }
  return g;
}

struct RopeLaunch {  // for rmsnorm_b200_last_plan
  RopePlan pl;
  char kind[16];
  unsigned x, y;
  int threads;
};

std::string describe_rope(const void* data) {
  const RopeLaunch& l = *static_cast<const RopeLaunch*>(data);
  char buf[128];
  std::snprintf(buf, sizeof(buf), "%s grid=%ux%u threads=%d lanes=%d jobs=%d+%d S=%d", l.kind, l.x, l.y, l.threads,
                1 << l.pl.lanes_shift, l.pl.jobs[0], l.pl.jobs[1], l.pl.S);
  return buf;
}

// Launches with programmatic dependent launch: the kernels wait for the one before them
// before their first global access.
template <typename Kernel>
int launch(UnitDevice* ud, Kernel kernel, const RopeGrid& g, cudaStream_t stream, const RopeParams& p,
           const char* kind) {
  const RopePlan& pl = g.pl;
  const dim3 grid = g.grid;
  const int threads = g.threads;
  {
    std::lock_guard<std::mutex> lock(ud->mu);
    const void* fn = reinterpret_cast<const void*>(kernel);
    if (!ud->attrs_done.count(fn)) {  // noted once it is done: a call that fails is made again
      if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRopeSmem) != cudaSuccess) {
        cudaGetLastError();
        return RMSNORM_B200_ERR_CUDA;
      }
      ud->attrs_done.insert(fn);
    }
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = g.smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, p, pl) != cudaSuccess) {
    cudaGetLastError();
    return RMSNORM_B200_ERR_CUDA;
  }
  RopeLaunch l = {pl, {}, grid.x, grid.y, threads};
  std::strncpy(l.kind, kind, sizeof(l.kind) - 1);
  return launched(describe_rope, l);
}

using RopeKernel = void (*)(const RopeParams, const RopePlan);

// One head a lane without a ring, or several with one.
template <typename T, int U>
RopeKernel pick_fwd(bool interleaved, bool norm) {
  constexpr bool kRing = U > 1;
  if (interleaved) return norm ? rope_fwd_kernel<T, U, true, true, kRing> : rope_fwd_kernel<T, U, true, false, kRing>;
  return norm ? rope_fwd_kernel<T, U, false, true, kRing> : rope_fwd_kernel<T, U, false, false, kRing>;
}

template <int U>
RopeKernel pick_fwd(const RopeParams& p) {
  if (p.dt == RMSNORM_B200_BF16) return pick_fwd<__nv_bfloat16, U>(p.interleaved, p.norm);
  return p.dt == RMSNORM_B200_F16 ? pick_fwd<__half, U>(p.interleaved, p.norm) : pick_fwd<float, U>(p.interleaved, p.norm);
}

template <typename T, int U, bool kPerHead>
RopeKernel pick_bwd(bool interleaved, bool norm) {
  constexpr int kBatch = kPerHead ? 2 : 1;
  if (interleaved)
    return norm ? rope_bwd_kernel<T, U, kBatch, true, true, kPerHead> : rope_bwd_kernel<T, U, kBatch, true, false, kPerHead>;
  return norm ? rope_bwd_kernel<T, U, kBatch, false, true, kPerHead> : rope_bwd_kernel<T, U, kBatch, false, false, kPerHead>;
}

// Heads a lane in the backward: two with sums for each of them.
constexpr int bwd_heads(bool per_head) { return per_head ? 2 : 4; }

template <bool kPerHead>
RopeKernel pick_bwd(const RopeParams& p) {
  constexpr int kHeads = bwd_heads(kPerHead);
  if (p.dt == RMSNORM_B200_BF16) return pick_bwd<__nv_bfloat16, kHeads, kPerHead>(p.interleaved, p.norm);
  return p.dt == RMSNORM_B200_F16 ? pick_bwd<__half, kHeads, kPerHead>(p.interleaved, p.norm)
                                  : pick_bwd<float, kHeads, kPerHead>(p.interleaved, p.norm);
}

int run_fwd(const rmsnorm_b200_rope_args* a, const rmsnorm_b200_rope_tensor* qo, const rmsnorm_b200_rope_tensor* ko,
            cudaStream_t stream) {
  int st = check(a);
  if (st) return st;
  if (!qo || !valid_tensor(*qo, a->tokens, a->q_heads) || (a->k_heads > 0 && (!ko || !valid_tensor(*ko, a->tokens, a->k_heads))))
    return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (a->tokens == 0) {
    rmsb_units::set_last_plan("rope fwd empty");
    return RMSNORM_B200_OK;
  }
  UnitDevice* ud = nullptr;
  st = unit_device(&ud);
  if (st) return st;
  Ranges ranges;
  add_ranges(ranges, a);
  add_tensor(ranges, *qo, a, a->q_heads);
  if (ko) add_tensor(ranges, *ko, a, a->k_heads);
  st = ranges.send(stream);
  if (st) return st;
  RopeParams p = params(a);
  p.out[0] = tensor(*qo);
  if (ko) p.out[1] = tensor(*ko);
  if (vectorised(a, {&a->q, &a->k, qo, ko})) {
    // Four heads a lane where that leaves every SM eight warps to run; single heads below.
    const bool apart = heads_apart(a->q, a->q_heads, a->head_dim) || heads_apart(a->k, a->k_heads, a->head_dim);
    RopeGrid g = plan(a, 4, 1, apart, ud->sm_count);
    const bool wide = a->tokens * (g.pl.jobs[0] + g.pl.jobs[1]) >= int64_t{8} * ud->sm_count;
    if (!wide) g = plan(a, 1, 0, false, ud->sm_count);
    return launch(ud, wide ? pick_fwd<4>(p) : pick_fwd<1>(p), g, stream, p, "rope_fwd");
  }
  const int64_t work = a->tokens * (a->q_heads + a->k_heads);
  const int64_t warps = kGenericThreads / 32;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>((work + warps - 1) / warps, int64_t{16} * ud->sm_count));
  rope_fwd_generic_kernel<<<grid, kGenericThreads, 0, stream>>>(p);
  return launched("rope_fwd_generic grid=" + std::to_string(grid));
}

struct BwdPlan {
  int64_t chunk = 1, chunks = 1;  // scalar kernel
  bool vec = false;
  bool per_head = false;          // partial rows of every head
  RopeGrid rope;
  int64_t rows = 0, width = 0;    // partial rows of dweight
};

int check_bwd(const rmsnorm_b200_rope_args* a, const rmsnorm_b200_rope_grads* g) {
  int st = check(a);
  if (st) return st;
  if (!g || !valid_tensor(g->dq_out, a->tokens, a->q_heads) || !valid_tensor(g->dk_out, a->tokens, a->k_heads) ||
      !valid_tensor(g->dq, a->tokens, a->q_heads) || !valid_tensor(g->dk, a->tokens, a->k_heads))
    return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if ((g->dq_weight && !a->q_weight) || (g->dk_weight && !a->k_weight)) return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  return RMSNORM_B200_OK;
}

BwdPlan plan_bwd(const UnitDevice* ud, const rmsnorm_b200_rope_args* a, const rmsnorm_b200_rope_grads* g) {
  BwdPlan pl;
  const int64_t heads = a->q_heads + a->k_heads;
  pl.per_head = (a->q_weight && a->q_weight_heads > 1) || (a->k_weight && a->k_weight_heads > 1);
  pl.vec = vectorised(a, {&a->q, &a->k, &g->dq_out, &g->dk_out, &g->dq, &g->dk});
  if (pl.vec) {
    bool apart = false;
    for (const auto* t : {&a->q, &g->dq_out}) apart = apart || heads_apart(*t, a->q_heads, a->head_dim);
    for (const auto* t : {&a->k, &g->dk_out}) apart = apart || heads_apart(*t, a->k_heads, a->head_dim);
    pl.rope = plan(a, bwd_heads(pl.per_head), 2, apart, ud->sm_count);
    const int64_t along = pl.rope.grid.x, across = pl.rope.grid.y;
    pl.rows = pl.per_head ? along : along * across;
    pl.width = (pl.per_head ? heads : 2) * a->head_dim;
    return pl;
  }
  pl.per_head = true;
  const int64_t target = std::max<int64_t>(1, (int64_t{16} * ud->sm_count + heads - 1) / heads);
  // at most 256 tokens per warp are added one after the other, at most 65535 chunks fit a grid
  pl.chunk = std::clamp<int64_t>((a->tokens + target - 1) / target, kGenericThreads / 32, 256 * (kGenericThreads / 32));
  pl.chunk = std::max<int64_t>(pl.chunk, (a->tokens + 65534) / 65535);
  pl.chunks = (a->tokens + pl.chunk - 1) / pl.chunk;
  pl.rows = pl.chunks;
  pl.width = heads * a->head_dim;
  return pl;
}

size_t workspace(const rmsnorm_b200_rope_grads* g, const BwdPlan& pl) {
  if (!g->dq_weight && !g->dk_weight) return 0;
  return static_cast<size_t>(pl.rows) * pl.width * sizeof(float);
}

int run_bwd(const rmsnorm_b200_rope_args* a, const rmsnorm_b200_rope_grads* g, void* ws, size_t ws_bytes,
            cudaStream_t stream) {
  int st = check_bwd(a, g);
  if (st) return st;
  UnitDevice* ud = nullptr;
  st = unit_device(&ud);
  if (st) return st;
  const BwdPlan pl = plan_bwd(ud, a, g);
  const size_t need = workspace(g, pl);
  if (need > ws_bytes || (need > 0 && (!ws || !aligned_to(ws, 16)))) return RMSNORM_B200_ERR_WORKSPACE;
  const int heads = a->q_heads + a->k_heads;
  Ranges ranges;
  if (a->tokens > 0) {
    add_ranges(ranges, a);
    add_tensor(ranges, g->dq_out, a, a->q_heads);
    add_tensor(ranges, g->dk_out, a, a->k_heads);
    add_tensor(ranges, g->dq, a, a->q_heads);
    add_tensor(ranges, g->dk, a, a->k_heads);
  }
  ranges.add(ws, need);
  const size_t wb = static_cast<size_t>(a->head_dim) * elem_bytes(a->weight_dtype);
  if (g->dq_weight) ranges.add(g->dq_weight, a->q_weight_heads * wb);
  if (g->dk_weight) ranges.add(g->dk_weight, a->k_weight_heads * wb);
  st = ranges.send(stream);
  if (st) return st;
  RopeParams p = params(a);
  p.dy[0] = tensor(g->dq_out); p.dy[1] = tensor(g->dk_out);
  p.out[0] = tensor(g->dq); p.out[1] = tensor(g->dk);
  p.part = need ? static_cast<float*>(ws) : nullptr;
  if (a->tokens > 0) {
    if (pl.vec) {
      st = launch(ud, pl.per_head ? pick_bwd<true>(p) : pick_bwd<false>(p), pl.rope, stream, p, "rope_bwd");
    } else {
      const dim3 grid(static_cast<unsigned>(heads), static_cast<unsigned>(pl.chunks));
      rope_bwd_generic_kernel<<<grid, kGenericThreads, 0, stream>>>(p, pl.chunk);
      st = launched("rope_bwd_generic chunks=" + std::to_string(pl.chunks));
    }
    if (st) return st;
  } else {
    rmsb_units::set_last_plan("rope bwd empty");
  }
  // the weights' gradients: fixed-order sums over the chunks (and over the heads that share
  // a weight), one launch for both
  ReduceParams rp = {};
  rp.C = a->tokens > 0 ? pl.rows : 0;
  rp.W = pl.width;
  rp.N = a->head_dim;
  int njobs = 0;
  int64_t blocks = 0;
  auto add_job = [&](int64_t first_head, void* out, int nheads, int w_heads) {
    ReduceJob& jb = rp.job[njobs++];
    jb.part = static_cast<const float*>(ws) + (pl.per_head ? first_head : first_head > 0) * a->head_dim;
    jb.out = out;
    jb.fold = pl.per_head && w_heads == 1 ? nheads : 1;
    jb.wout = static_cast<int64_t>(w_heads) * a->head_dim;
    jb.out_dt = a->weight_dtype;
    const int64_t cols = reduce_vectorised(jb, rp.W) ? kReduceVCols : kReduceCols;
    blocks = std::max(blocks, (jb.wout + cols - 1) / cols);
  };
  if (g->dq_weight) add_job(0, g->dq_weight, a->q_heads, a->q_weight_heads);
  if (g->dk_weight) add_job(a->q_heads, g->dk_weight, a->k_heads, a->k_weight_heads);
  if (njobs == 0) return RMSNORM_B200_OK;
  reduce_partials_kernel<<<dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(njobs)), kReduceThreads, 0,
                           stream>>>(rp);
  return launched("");
}

int workspace_size(const rmsnorm_b200_rope_args* a, const rmsnorm_b200_rope_grads* g, size_t* bytes) {
  if (!bytes) return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  *bytes = 0;
  int st = check_bwd(a, g);
  if (st) return st;
  UnitDevice* ud = nullptr;
  st = unit_device(&ud);
  if (st) return st;
  *bytes = workspace(g, plan_bwd(ud, a, g));
  return RMSNORM_B200_OK;
}

}  // namespace
}  // namespace rmsb200

using namespace rmsb200;

extern "C" int rmsnorm_b200_rope_fwd(const rmsnorm_b200_rope_args* a, const rmsnorm_b200_rope_tensor* q_out,
                                     const rmsnorm_b200_rope_tensor* k_out, void* stream) {
  return entry([&] { return run_fwd(a, q_out, k_out, static_cast<cudaStream_t>(stream)); });
}

extern "C" int rmsnorm_b200_rope_bwd_workspace_size(const rmsnorm_b200_rope_args* a,
                                                    const rmsnorm_b200_rope_grads* g, size_t* bytes) {
  return entry([&] { return workspace_size(a, g, bytes); });
}

extern "C" int rmsnorm_b200_rope_bwd(const rmsnorm_b200_rope_args* a, const rmsnorm_b200_rope_grads* g,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  return entry([&] { return run_bwd(a, g, workspace, workspace_bytes, static_cast<cudaStream_t>(stream)); });
}
