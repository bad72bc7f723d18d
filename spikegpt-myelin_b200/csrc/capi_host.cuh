// Host-side pieces shared by the translation units behind the C ABI: the
// thread's last error, launch accounting and per-kernel timing, and small
// argument helpers. One copy per process (inline variables).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <mutex>
#include <utility>
#include <vector>

#include "spikegpt_wkv.h"

namespace wkv_host {

inline thread_local char g_last_error[512] = "";

// ------------------------------------------------ launch accounting / timing
//
// Every kernel launch goes through launch(): it bumps a per-kind counter and,
// while timing is enabled, brackets the launch with CUDA events recorded on the
// launch stream, so per-kernel device time can be read back by the caller.

enum Kind {
  K_FWD_Y, K_FWD_STATE, K_BWD_GRAD, K_BWD_ADJ, K_CARRY_FWD, K_CARRY_ADJ, K_STEP, K_LIF_FWD, K_LIF_BWD,
  K_MIX_FWD, K_MIX_BWD, K_MIX_RED,
  K_GATE_FWD, K_GATE_BWD, K_RSQ_FWD, K_RSQ_BWD, K_RESID, K_LIF_SUM, K_R7_FWD, K_XENT_FWD, K_XENT_BWD,
  K_CONV_FWD, K_CONV_BWD, K_CONV_STEP, K_SCAN_SUM, K_SCAN_FWD, K_SCAN_ADJ, K_SCAN_BWD, K_SCAN_RED, K_SCAN_STEP,
  K_LN_FWD, K_LN_BWD, K_COL_SUM, K_Q4,
  K_COUNT
};
inline const char* const kKindNames[K_COUNT] = {
    "wkv_fwd_kernel<y>",      "wkv_fwd_kernel<state>", "wkv_bwd_kernel<grad>",
    "wkv_bwd_kernel<adjoint>", "wkv_carry_fwd_kernel",  "wkv_carry_adj_kernel",
    "wkv_step_kernel",        "lif_fwd_kernel",        "lif_bwd_kernel",
    "ln_mix_fwd_kernel",      "ln_mix_bwd_kernel",     "ln_mix_reduce_kernel",
    "gate_fwd_kernel",        "gate_bwd_kernel",       "relu_square_fwd_kernel",
    "relu_square_bwd_kernel", "residual_add_kernel",   "lif_bwd_summary_kernel",
    "rwkv7_fwd_kernel",       "xent_fwd_kernel",       "xent_bwd_kernel",
    "causal_conv_fwd_kernel", "causal_conv_bwd_kernel", "causal_conv_step_kernel",
    "scan_summary_kernel",   "scan_fwd_kernel",       "scan_adjoint_kernel",
    "scan_bwd_kernel",       "scan_reduce_kernel",    "scan_step_kernel",
    "layer_norm_fwd_kernel", "layer_norm_bwd_kernel", "column_sum_kernel",
    "q4_matvec_kernel"};

inline std::atomic<long long> g_launches[K_COUNT];
inline std::atomic<bool> g_timing{false};
inline std::mutex g_timing_mu;
struct TimedLaunch {
  int kind;
  cudaEvent_t start, stop;
};
inline std::vector<TimedLaunch> g_timed;
inline std::vector<cudaEvent_t> g_event_pool;

inline cudaEvent_t pooled_event() {
  std::lock_guard<std::mutex> lk(g_timing_mu);
  if (!g_event_pool.empty()) {
    cudaEvent_t e = g_event_pool.back();
    g_event_pool.pop_back();
    return e;
  }
  cudaEvent_t e = nullptr;
  if (cudaEventCreate(&e) != cudaSuccess) return nullptr;
  return e;
}

template <class F>
void launch(int kind, cudaStream_t st, F&& f) {
  g_launches[kind].fetch_add(1, std::memory_order_relaxed);
  if (!g_timing.load(std::memory_order_relaxed)) {
    f();
    return;
  }
  cudaEvent_t a = pooled_event(), b = pooled_event();
  if (a) cudaEventRecord(a, st);
  f();
  if (b) cudaEventRecord(b, st);
  if (a && b) {
    std::lock_guard<std::mutex> lk(g_timing_mu);
    g_timed.push_back(TimedLaunch{kind, a, b});
  }
}

inline int fail(int status, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_last_error, sizeof(g_last_error), fmt, ap);
  va_end(ap);
  return status;
}

inline int cuda_fail(cudaError_t e, const char* what) {
  return fail(WKV_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

inline size_t dtype_size(int dtype) {
  switch (dtype) {
    case WKV_DTYPE_F32: return 4;
    case WKV_DTYPE_BF16: return 2;
    case WKV_DTYPE_F16: return 2;
    default: return 0;
  }
}

inline int sm_count() {
  static int cached[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (cached[dev] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0)
      n = 148;
    cached[dev] = n;
  }
  return cached[dev];
}

inline int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? WKV_OK : cuda_fail(e, what);
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

constexpr size_t kAlign = 256;
inline size_t round_up(size_t x) { return (x + kAlign - 1) / kAlign * kAlign; }

// Kernels whose dynamic shared memory exceeds the 48 KB default (less 2 KB for static
// arrays) opt in once per device.
template <typename K>
cudaError_t allow_smem(K* kernel, size_t bytes) {
  if (bytes <= 46 * 1024) return cudaSuccess;
  static std::mutex mu;
  static std::vector<std::pair<const void*, int>> done;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> lk(mu);
  for (auto& d : done)
    if (d.first == reinterpret_cast<const void*>(kernel) && d.second == dev) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess) done.emplace_back(reinterpret_cast<const void*>(kernel), dev);
  return e;
}

}  // namespace wkv_host
