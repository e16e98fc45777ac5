// kv_cache.cu -- rmsnorm_b200_cache_write and rmsnorm_b200_cache_read: argument checks and launch.
#define RMSB_UNIT kv_cache
#include "unit_state.cuh"

#include "kv_cache_kernels.cuh"

namespace rmsb200 {
namespace {

using CacheKernel = void (*)(const CacheParams);

int check(const rmsnorm_b200_cache_args* c) {
  if (!c || c->pages < 0 || c->pages >= (int64_t{1} << 31) || c->page_size < 1 || c->heads < 1 ||
      c->heads > RMSNORM_B200_ROPE_MAX_HEADS || c->head_dim < 1 || c->head_dim > RMSNORM_B200_ROPE_MAX_HEAD_DIM)
    return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (c->cache_dtype != RMSNORM_B200_E4M3 && c->cache_dtype != RMSNORM_B200_I8) return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  for (const rmsnorm_b200_cache_tensor* t : {&c->k, &c->v}) {
    if (c->pages > 0 && (!t->data || !t->scales)) return RMSNORM_B200_ERR_INVALID_ARGUMENT;
    if (t->page_stride < 0 || t->slot_stride < 0 || t->head_stride < 0 || t->scale_page_stride < 0 ||
        t->scale_slot_stride < 0 || t->scale_head_stride < 0)
      return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  }
  return RMSNORM_B200_OK;
}

CacheSide side_of(const rmsnorm_b200_cache_args* c, const rmsnorm_b200_cache_tensor& t, void* x, int64_t x_token,
                  int64_t x_head, int x_bytes) {
  CacheSide s = {};
  s.data = static_cast<unsigned char*>(t.data);
  s.page = t.page_stride; s.slot = t.slot_stride; s.head = t.head_stride;
  s.scales = t.scales;
  s.s_page = t.scale_page_stride; s.s_slot = t.scale_slot_stride; s.s_head = t.scale_head_stride;
  s.x = x; s.x_token = x_token; s.x_head = x_head;
  const bool whole = c->head_dim % 8 == 0;
  s.vec_x = whole && aligned_to(x, 16) && x_token * x_bytes % 16 == 0 && x_head * x_bytes % 16 == 0;
  s.vec_q = whole && aligned_to(t.data, 8) && t.page_stride % 8 == 0 && t.slot_stride % 8 == 0 && t.head_stride % 8 == 0;
  return s;
}

void add_ranges(Ranges* r, const rmsnorm_b200_cache_args* c, const CacheSide& s, int64_t tokens, int x_bytes) {
  if (c->pages > 0) {
    r->add(s.data, (c->pages - 1) * s.page + (c->page_size - 1) * s.slot + (c->heads - 1) * s.head + c->head_dim);
    r->add(s.scales, ((c->pages - 1) * s.s_page + (c->page_size - 1) * s.s_slot + (c->heads - 1) * s.s_head + 1) * 4);
  }
  r->add(s.x, ((tokens - 1) * s.x_token + (c->heads - 1) * s.x_head + c->head_dim) * x_bytes);
}

void set_sizes(CacheParams* p, const rmsnorm_b200_cache_args* c) {
  constexpr int64_t kMost = int64_t{1} << 31;
  p->page_size = c->page_size;
  p->heads = c->heads;
  p->head_dim = c->head_dim;
  p->by_page = divisor_of(static_cast<uint32_t>(c->page_size));
  p->small = p->tokens < kMost / c->heads && c->pages < kMost / c->page_size;  // there are no more rounds than heads
}

// Lanes of a head with one octet of columns each; where a lane has two, a head takes half of them.
template <bool kWrite, typename X, typename Q, int kItems, int kOctets>
CacheKernel pick_lanes(int lanes) {
  if constexpr (kWrite)
    return lanes == 8    ? cache_write_kernel<X, Q, 8 / kOctets, kItems, kOctets>
           : lanes == 16 ? cache_write_kernel<X, Q, 16 / kOctets, kItems, kOctets>
                         : cache_write_kernel<X, Q, 32 / kOctets, kItems, kOctets>;
  else
    return lanes == 8    ? cache_read_kernel<X, Q, 8, kItems>
           : lanes == 16 ? cache_read_kernel<X, Q, 16, kItems>
                         : cache_read_kernel<X, Q, 32, kItems>;
}

template <bool kWrite, typename X>
CacheKernel pick(int cache_dtype, int lanes, int items, int octets) {
  constexpr int kMost = kWrite && sizeof(X) == 2 ? 2 : 1;
  if (cache_dtype == RMSNORM_B200_E4M3)
    return items == 1    ? pick_lanes<kWrite, X, E4M3, 1, 1>(lanes)
           : octets == 1 ? pick_lanes<kWrite, X, E4M3, 4, 1>(lanes)
                         : pick_lanes<kWrite, X, E4M3, 4, kMost>(lanes);
  return items == 1    ? pick_lanes<kWrite, X, I8, 1, 1>(lanes)
         : octets == 1 ? pick_lanes<kWrite, X, I8, 4, 1>(lanes)
                       : pick_lanes<kWrite, X, I8, 4, kMost>(lanes);
}

struct CacheLaunch {
  const char* kind;
  unsigned grid;
  int lanes, items;
};

std::string describe(const void* data) {
  const CacheLaunch& l = *static_cast<const CacheLaunch*>(data);
  char buf[96];
  std::snprintf(buf, sizeof(buf), "%s grid=%u lanes=%d items=%d", l.kind, l.grid, l.lanes, l.items);
  return buf;
}

template <bool kWrite>
int launch(UnitDevice* ud, const rmsnorm_b200_cache_args* c, CacheParams& p, int dtype, cudaStream_t stream) {
  const int lanes = c->head_dim <= 64 ? 8 : c->head_dim <= 128 ? 16 : 32;
  // Four heads of a token in flight a lane, and two octets of each when 16-bit values are written
  // (4 registers an octet), where it has that many and that leaves two CTAs for every SM.
  const auto enough = [&](int n) { return p.tokens * p.heads * lanes >= int64_t{2} * n * kCacheThreads * ud->sm_count; };
  const int octets = kWrite && dtype != RMSNORM_B200_F32 && c->heads >= 3 && enough(8) ? 2 : 1;
  const int each = c->heads >= 3 && enough(4) ? 4 : 1;
  p.rounds = (c->heads + each - 1) / each;
  p.by_rounds = divisor_of(static_cast<uint32_t>(p.rounds));
  const int64_t per = kCacheThreads / (lanes / octets), grid = (p.tokens * p.rounds + per - 1) / per;
  if (grid >= int64_t{1} << 31) return RMSNORM_B200_ERR_UNSUPPORTED;
  const CacheKernel kernel = dtype == RMSNORM_B200_F32    ? pick<kWrite, float>(c->cache_dtype, lanes, each, octets)
                             : dtype == RMSNORM_B200_BF16 ? pick<kWrite, __nv_bfloat16>(c->cache_dtype, lanes, each, octets)
                                                          : pick<kWrite, __half>(c->cache_dtype, lanes, each, octets);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid), kWrite ? 2 : 1);
  cfg.blockDim = dim3(kCacheThreads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, p) != cudaSuccess) {
    cudaGetLastError();
    return RMSNORM_B200_ERR_CUDA;
  }
  const CacheLaunch l = {kWrite ? "cache_write" : "cache_read", static_cast<unsigned>(grid), lanes / octets, each};
  return launched(describe, l);
}

int write(const rmsnorm_b200_cache_args* c, const rmsnorm_b200_cache_write_args* a, cudaStream_t stream) {
  int st = check(c);
  if (st) return st;
  if (!a || a->tokens < 0 || !valid_dt(a->dtype)) return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  for (const rmsnorm_b200_rope_tensor* t : {&a->k, &a->v})
    if (a->tokens > 0 && (!t->data || t->token_stride < 0 || t->head_stride < 0)) return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (a->tokens > 0 && !a->slots) return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (a->tokens >= int64_t{1} << 40) return RMSNORM_B200_ERR_UNSUPPORTED;
  if (a->tokens == 0) {
    rmsb_units::set_last_plan("cache_write empty");
    return RMSNORM_B200_OK;
  }
  UnitDevice* ud = nullptr;
  st = unit_device(&ud);
  if (st) return st;
  const int xb = elem_bytes(a->dtype);
  CacheParams p = {};
  p.side[0] = side_of(c, c->k, a->k.data, a->k.token_stride, a->k.head_stride, xb);
  p.side[1] = side_of(c, c->v, a->v.data, a->v.token_stride, a->v.head_stride, xb);
  p.pages = c->pages; p.tokens = a->tokens;
  p.slots = a->slots; p.slots_64bit = a->slots_64bit != 0;
  set_sizes(&p, c);
  Ranges ranges;
  for (const CacheSide& s : p.side) add_ranges(&ranges, c, s, a->tokens, xb);
  ranges.add(a->slots, a->tokens * (p.slots_64bit ? 8 : 4));
  st = ranges.send(stream);
  if (st) return st;
  return launch<true>(ud, c, p, a->dtype, stream);
}

int read(const rmsnorm_b200_cache_args* c, const rmsnorm_b200_cache_read_args* a, cudaStream_t stream) {
  int st = check(c);
  if (st) return st;
  if (!a || a->tokens < 0 || a->sequences < 0 || a->sequences >= (int64_t{1} << 31) || a->table_width < 0 ||
      a->table_stride < 0 || !valid_dt(a->dtype))
    return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (a->tokens > 0 && (!a->starts || !a->k || !a->v || (a->sequences > 0 && a->table_width > 0 && !a->page_table)))
    return RMSNORM_B200_ERR_INVALID_ARGUMENT;
  if (a->tokens >= int64_t{1} << 40) return RMSNORM_B200_ERR_UNSUPPORTED;
  if (a->tokens == 0) {
    rmsb_units::set_last_plan("cache_read empty");
    return RMSNORM_B200_OK;
  }
  UnitDevice* ud = nullptr;
  st = unit_device(&ud);
  if (st) return st;
  const int xb = elem_bytes(a->dtype);
  const int64_t row = static_cast<int64_t>(c->heads) * c->head_dim;
  CacheParams p = {};
  p.side[0] = side_of(c, c->k, a->k, row, c->head_dim, xb);
  p.side[1] = side_of(c, c->v, a->v, row, c->head_dim, xb);
  p.pages = c->pages; p.tokens = a->tokens;
  p.table = a->page_table; p.starts = a->starts;
  p.table_width = a->table_width; p.table_stride = a->table_stride;
  p.sequences = static_cast<int32_t>(a->sequences);
  p.zero_rest = a->zero_rest != 0;
  set_sizes(&p, c);
  Ranges ranges;
  for (const CacheSide& s : p.side) add_ranges(&ranges, c, s, a->tokens, xb);
  ranges.add(a->starts, (a->sequences + 1) * 4);
  if (a->sequences > 0 && a->table_width > 0)
    ranges.add(a->page_table, ((a->sequences - 1) * a->table_stride + a->table_width) * 4);
  st = ranges.send(stream);
  if (st) return st;
  return launch<false>(ud, c, p, a->dtype, stream);
}

}  // namespace
}  // namespace rmsb200

using namespace rmsb200;

extern "C" int rmsnorm_b200_cache_write(const rmsnorm_b200_cache_args* c, const rmsnorm_b200_cache_write_args* a,
                                        void* stream) {
  return entry([&] { return write(c, a, static_cast<cudaStream_t>(stream)); });
}

extern "C" int rmsnorm_b200_cache_read(const rmsnorm_b200_cache_args* c, const rmsnorm_b200_cache_read_args* a,
                                       void* stream) {
  return entry([&] { return read(c, a, static_cast<cudaStream_t>(stream)); });
}
