// generic_kernels.cuh -- kernels for every case the streaming kernels do not take:
// hidden sizes that are not a multiple of 8, pointers that are not 16-byte aligned,
// dtype combinations outside the specialised set, per-head segments whose length is not
// a power of two <= 32 vectors, and rows too long for the cluster split. They compute
// the same fp32 math with scalar runtime-typed loads (one CTA per row, grid-stride) and
// keep dweight/dbias deterministic with fixed-order chunked column sums.
#pragma once

#include "column_sums.cuh"

namespace rmsb200 {

struct GenFwdParams {
  int64_t rows, N;
  int32_t H;
  const void* x; int32_t x_dt;
  const void* res; int32_t res_dt;
  const void* w; int32_t w_dt, w_ph;
  const void* b; int32_t b_dt, b_ph;
  void* out; int32_t out_dt;
  void* ro; int32_t ro_dt;
  float* rstd;
  float eps;
};

__global__ void __launch_bounds__(kGenericThreads) fwd_generic_kernel(const GenFwdParams p) {
  __shared__ float red[32];
  const int64_t N = p.N;
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const int64_t base = r * N;
    const int64_t head = r % p.H;
    float acc = 0.f;
    for (int64_t n = threadIdx.x; n < N; n += blockDim.x) {
      float v = load1_rt(p.x, p.x_dt, base + n);
      if (p.res) v += load1_rt(p.res, p.res_dt, base + n);
      acc = fmaf(v, v, acc);
    }
    acc = block_sum_fixed(acc, red);
    const float rs = rsqrtf(acc / static_cast<float>(N) + p.eps);
    for (int64_t n = threadIdx.x; n < N; n += blockDim.x) {
      float v = load1_rt(p.x, p.x_dt, base + n);
      if (p.res) v += load1_rt(p.res, p.res_dt, base + n);
      if (p.ro) store1_rt(p.ro, p.ro_dt, base + n, v);
      const float w = p.w ? load1_rt(p.w, p.w_dt, (p.w_ph ? head * N : 0) + n) : 1.f;
      const float b = p.b ? load1_rt(p.b, p.b_dt, (p.b_ph ? head * N : 0) + n) : 0.f;
      store1_rt(p.out, p.out_dt, base + n, fmaf(v * rs, w, b));
    }
    if (threadIdx.x == 0 && p.rstd) st1(&p.rstd[r], rs);
  }
}

// LayerNorm forward, generic path: mean, then the mean of squared deviations (two passes,
// so the variance has no cancellation), then out = (x - mean) * rstd * w + b. `out` may be
// null (statistics only); w null = ones, b null = zeros.
struct GenLnParams {
  int64_t rows, N;
  const void* x; int32_t x_dt;
  const void* w; int32_t w_dt;
  const void* b; int32_t b_dt;
  void* out; int32_t out_dt;
  float* mean;
  float* rstd;
  float eps;
};

__global__ void __launch_bounds__(kGenericThreads) ln_generic_kernel(const GenLnParams p) {
  __shared__ float red[32];
  const int64_t N = p.N;
  const float inv_n = 1.f / static_cast<float>(N);
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const int64_t base = r * N;
    float acc = 0.f;
    for (int64_t n = threadIdx.x; n < N; n += blockDim.x) acc += load1_rt(p.x, p.x_dt, base + n);
    const float mean = block_sum_fixed(acc, red) * inv_n;
    acc = 0.f;
    for (int64_t n = threadIdx.x; n < N; n += blockDim.x) {
      const float d = load1_rt(p.x, p.x_dt, base + n) - mean;
      acc = fmaf(d, d, acc);
    }
    const float rs = rsqrtf(fmaf(block_sum_fixed(acc, red), inv_n, p.eps));
    if (p.out) {
      for (int64_t n = threadIdx.x; n < N; n += blockDim.x) {
        const float d = load1_rt(p.x, p.x_dt, base + n) - mean;
        const float w = p.w ? load1_rt(p.w, p.w_dt, n) : 1.f;
        const float b = p.b ? load1_rt(p.b, p.b_dt, n) : 0.f;
        store1_rt(p.out, p.out_dt, base + n, fmaf(d * rs, w, b));
      }
    }
    if (threadIdx.x == 0) {
      if (p.mean) st1(&p.mean[r], mean);
      if (p.rstd) st1(&p.rstd[r], rs);
    }
  }
}

__global__ void __launch_bounds__(kGenericThreads) bwd_generic_dx_kernel(const GenBwdParams p) {
  __shared__ float red[32];
  const int64_t N = p.N;
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const int64_t base = r * N;
    const int64_t woff = p.w_ph ? (r % p.H) * N : 0;
    const float rs = ld1(&p.rstd[r]);
    float acc = 0.f;
    for (int64_t n = threadIdx.x; n < N; n += blockDim.x) {
      const float xh = load1_rt(p.x, p.x_dt, base + n) * rs;
      const float w = p.w ? load1_rt(p.w, p.w_dt, woff + n) : 1.f;
      acc = fmaf(xh, load1_rt(p.dy, p.dy_dt, base + n) * w, acc);
    }
    acc = block_sum_fixed(acc, red);
    const float c = acc / static_cast<float>(N);
    for (int64_t n = threadIdx.x; n < N; n += blockDim.x) {
      const float xh = load1_rt(p.x, p.x_dt, base + n) * rs;
      const float w = p.w ? load1_rt(p.w, p.w_dt, woff + n) : 1.f;
      float g = (load1_rt(p.dy, p.dy_dt, base + n) * w - xh * c) * rs;
      if (p.dro) g += load1_rt(p.dro, p.dro_dt, base + n);
      store1_rt(p.dx, p.dx_dt, base + n, g);
      if (p.dres) store1_rt(p.dres, p.dres_dt, base + n, g);
    }
  }
}

// Failure-detection self test: one CTA waits on an mbarrier that nothing arrives at.
__global__ void selftest_wait_kernel(unsigned long long timeout_ns) {
  __shared__ __align__(8) uint64_t bar;
  if (threadIdx.x == 0) {
    mbar_init(&bar, 1);
    fence_mbar_init();
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait(&bar, 0)) {
      if (globaltimer_ns() - t0 > timeout_ns) {
        record_error(RMSNORM_B200_ERR_DEVICE_TIMEOUT, kSiteSelftest);
        break;
      }
    }
  }
}

}  // namespace rmsb200
