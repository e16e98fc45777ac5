// unit_state.cuh -- host-side state and launch helpers of a translation unit other than the
// main one: per-device properties, kernel attributes, the hooks of translation_units.h and
// (bounds-checked build) the registration of a call's byte ranges.
//
// Include it after defining RMSB_UNIT (fused_fwd, fused_bwd, rope, block_quant, block_mm, kv_cache): the kernels and device
// variables of the shared headers then live in a namespace of that unit, so that the units
// link into one library.
#pragma once

#ifndef RMSB_UNIT
#error "RMSB_UNIT names the translation unit"
#endif
#define RMSB_CAT2(a, b) a##b
#define RMSB_CAT(a, b) RMSB_CAT2(a, b)
#define rmsb200 RMSB_CAT(rmsb200_, RMSB_UNIT)

#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <memory>
#include <mutex>
#include <string>
#include <tuple>
#include <unordered_set>
#include <vector>

#include "device_common.cuh"
#include "translation_units.h"

namespace rmsb200 {
namespace {

constexpr int kSmemOptIn = 232448;  // largest dynamic shared memory of a CTA (227 KB)

int elem_bytes(int dt) { return dt == RMSNORM_B200_F32 ? 4 : 2; }
bool valid_dt(int dt) { return dt == RMSNORM_B200_F16 || dt == RMSNORM_B200_BF16 || dt == RMSNORM_B200_F32; }
bool aligned_to(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

struct UnitDevice {
  int sm_count = 0;
  std::mutex mu;
  std::unordered_set<const void*> attrs_done;
  std::map<std::tuple<const void*, int, int>, int> clusters;  // that fit, by kernel, CTAs and shared memory
};

std::mutex g_unit_mu;
std::vector<std::unique_ptr<UnitDevice>> g_unit_devices;

int unit_device(UnitDevice** out) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return RMSNORM_B200_ERR_NO_DEVICE;
  std::lock_guard<std::mutex> lock(g_unit_mu);
  if (static_cast<int>(g_unit_devices.size()) <= dev) g_unit_devices.resize(dev + 1);
  if (!g_unit_devices[dev]) {
    auto st = std::make_unique<UnitDevice>();
    if (cudaDeviceGetAttribute(&st->sm_count, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
      return RMSNORM_B200_ERR_NO_DEVICE;
    g_unit_devices[dev] = std::move(st);
  }
  *out = g_unit_devices[dev].get();
  return RMSNORM_B200_OK;
}

#ifdef RMSB_DEBUG_BOUNDS
// The byte ranges the kernels of one call may access, written to the device on the call's
// stream before its first launch.
struct Ranges {
  DbgRanges r{};
  void add(const void* p, size_t bytes) {
    if (!p || bytes == 0 || r.n >= kDbgMaxRanges) return;
    r.lo[r.n] = reinterpret_cast<uintptr_t>(p);
    r.hi[r.n] = r.lo[r.n] + bytes;
    ++r.n;
  }
  // Self test of the checker: RMSNORM_B200_DEBUG_CLIP_OUT=k registers an output k bytes short.
  void add_out(const void* p, size_t bytes) {
    const char* v = std::getenv("RMSNORM_B200_DEBUG_CLIP_OUT");
    const size_t clip = v ? static_cast<size_t>(std::atoi(v)) : 0;
    add(p, clip < bytes ? bytes - clip : bytes);
  }
  int send(cudaStream_t stream) {
    dbg_ranges_kernel<<<1, 32, 0, stream>>>(r);
    return cudaGetLastError() == cudaSuccess ? RMSNORM_B200_OK : RMSNORM_B200_ERR_CUDA;
  }
};
#else
struct Ranges {
  void add(const void*, size_t) {}
  void add_out(const void*, size_t) {}
  int send(cudaStream_t) { return RMSNORM_B200_OK; }
};
#endif

int unit_status(cudaStream_t s, rmsb_units::UnitStatus* words, bool clear) {
  if (cudaMemcpyFromSymbolAsync(&words->status, g_status, sizeof(int), 0, cudaMemcpyDeviceToHost, s) != cudaSuccess ||
      cudaMemcpyFromSymbolAsync(&words->where, g_status_where, sizeof(int), 0, cudaMemcpyDeviceToHost, s) !=
          cudaSuccess ||
      cudaMemcpyFromSymbolAsync(&words->data_status, g_data_status, sizeof(int), 0, cudaMemcpyDeviceToHost, s) !=
          cudaSuccess ||
      cudaMemcpyFromSymbolAsync(&words->data_where, g_data_status_where, sizeof(int), 0, cudaMemcpyDeviceToHost, s) !=
          cudaSuccess)
    return RMSNORM_B200_ERR_CUDA;
  if (clear) {
    static const int zero = 0;
    if (cudaMemcpyToSymbolAsync(g_status, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, s) != cudaSuccess ||
        cudaMemcpyToSymbolAsync(g_status_where, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, s) != cudaSuccess ||
        cudaMemcpyToSymbolAsync(g_data_status, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, s) != cudaSuccess ||
        cudaMemcpyToSymbolAsync(g_data_status_where, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, s) != cudaSuccess)
      return RMSNORM_B200_ERR_CUDA;
  }
  return RMSNORM_B200_OK;
}

int unit_set_wait_timeout(unsigned long long ns) {
  return cudaMemcpyToSymbol(g_wait_timeout_ns, &ns, sizeof(ns)) == cudaSuccess ? RMSNORM_B200_OK
                                                                               : RMSNORM_B200_ERR_CUDA;
}

int unit_report(unsigned long long (&words)[4], bool clear) {
#ifdef RMSB_DEBUG_BOUNDS
  if (cudaMemcpyFromSymbol(words, g_dbg_report, sizeof(words)) != cudaSuccess) return RMSNORM_B200_ERR_CUDA;
  if (clear) {
    const unsigned long long z[4] = {0, 0, 0, 0};
    if (cudaMemcpyToSymbol(g_dbg_report, z, sizeof(z)) != cudaSuccess) return RMSNORM_B200_ERR_CUDA;
  }
  return RMSNORM_B200_OK;
#else
  (void)words;
  (void)clear;
  return RMSNORM_B200_ERR_UNSUPPORTED;
#endif
}

// The status of the launch just made; counts it and records the plan's description.
int launched(std::string plan, uint64_t n = 1) {
  if (cudaGetLastError() != cudaSuccess) return RMSNORM_B200_ERR_CUDA;
  rmsb_units::count_launches(n);
  if (!plan.empty()) rmsb_units::set_last_plan(std::move(plan));
  return RMSNORM_B200_OK;
}

// The same with a plan whose text is made on demand.
template <typename Plan>
int launched(rmsb_units::PlanText make, const Plan& plan) {
  static_assert(sizeof(Plan) <= rmsb_units::kPlanBytes, "plan size");
  if (cudaGetLastError() != cudaSuccess) return RMSNORM_B200_ERR_CUDA;
  rmsb_units::count_launches(1);
  rmsb_units::set_last_plan(make, &plan, sizeof(plan));
  return RMSNORM_B200_OK;
}

// The body of a C entry: no exception leaves the library (what can throw here is the host's
// memory running out).
template <typename Body>
int entry(Body&& body) noexcept {
  try {
    return body();
  } catch (...) {
    return RMSNORM_B200_ERR_CUDA;
  }
}

}  // namespace
}  // namespace rmsb200

namespace rmsb_units {
const UnitHooks RMSB_CAT(RMSB_UNIT, _unit) = {rmsb200::unit_status, rmsb200::unit_set_wait_timeout,
                                              rmsb200::unit_report};
}  // namespace rmsb_units
