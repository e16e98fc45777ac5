// translation_units.h -- what the library's translation units share on the host.
//
// The library is compiled from several translation units without relocatable device code,
// so each has its own copy of the device-side state that device_common.cuh defines (status
// word, wait limit, bounds-check report). The main unit (rmsnorm_b200.cu) owns the C entry
// points that read and set that state; every other unit hands it a UnitHooks.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>
#include <string>

namespace rmsb_units {

// A unit's status words: a wait that ran out, and a value among a call's data.
struct UnitStatus {
  int status = 0, where = 0;
  int data_status = 0, data_where = 0;
};

struct UnitHooks {
  // Enqueues the read (and clear) of the unit's status words; the caller synchronises.
  int (*status)(cudaStream_t stream, UnitStatus* words, bool clear);
  int (*set_wait_timeout)(unsigned long long ns);
  // The four words of the unit's bounds-check report (bounds-checked build only).
  int (*report)(unsigned long long (&words)[4], bool clear);
};

extern const UnitHooks fused_fwd_unit;
extern const UnitHooks fused_bwd_unit;
extern const UnitHooks rope_unit;

// Bookkeeping of the main unit: rmsnorm_b200_launch_count and rmsnorm_b200_last_plan.
void count_launches(uint64_t n);
void set_last_plan(std::string plan);

// The same, as the function that makes the text from a copy of `data` (at most kPlanBytes).
using PlanText = std::string (*)(const void* data);
constexpr size_t kPlanBytes = 256;
void set_last_plan(PlanText make, const void* data, size_t bytes);

}  // namespace rmsb_units
