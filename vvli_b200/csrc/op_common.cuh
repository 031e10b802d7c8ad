// op_common.cuh - host-side checks shared by the context-free operators of the paged serving step.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <exception>
#include <mutex>
#include <string>

#include "../../include/vvli_cuda.h"

namespace vvli {
void set_last_error(const std::string& what);  // runtime.cu

inline bool aligned_to(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Makes `device` current and puts the caller's device back.
struct OpDeviceGuard {
  int prev = -1;
  cudaError_t enter(int device) {
    cudaError_t e = cudaGetDevice(&prev);
    if (e == cudaSuccess && prev == device) {
      prev = -1;
      return e;
    }
    return e == cudaSuccess ? cudaSetDevice(device) : e;
  }
  ~OpDeviceGuard() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

// One C entry: `check` gives the reason an argument is refused (or ""),
// before any CUDA call; `queue` launches with `device` current.  No exception
// leaves it.
template <class Check, class Queue>
int run_op(const char* name, int device, Check check, Queue queue) noexcept {
  try {
    const std::string bad = check();
    if (!bad.empty()) {
      set_last_error(std::string(name) + ": " + bad);
      return VVLI_ERR_INVALID_ARGUMENT;
    }
    OpDeviceGuard guard;
    cudaError_t e = guard.enter(device);
    if (e == cudaSuccess) e = queue();
    if (e != cudaSuccess) {
      cudaGetLastError();  // a refused launch must not surface in the caller's next call
      set_last_error(std::string(name) + ": " + cudaGetErrorString(e));
      return VVLI_ERR_CUDA;
    }
    return VVLI_OK;
  } catch (...) {  // out of host memory
    return VVLI_ERR_OOM;
  }
}

// "" when page_size is one the kernels take.
inline std::string check_page_size(uint64_t p) {
  return p == 16 || p == 32 || p == 64 || p == 128 ? "" : "page_size must be 16, 32, 64 or 128";
}

constexpr int kOpMaxDevices = 64;

// What an operator does once per device.  Only success is kept: a setup that
// failed (out of memory, say) is tried again by the next call.
class SetupOnce {
  std::atomic<bool> done_{false};
  std::mutex mutex_;

 public:
  template <class Setup>
  cudaError_t operator()(Setup setup) {
    if (done_.load(std::memory_order_acquire)) return cudaSuccess;
    std::lock_guard<std::mutex> lock(mutex_);
    if (done_.load(std::memory_order_relaxed)) return cudaSuccess;
    const cudaError_t e = setup();
    if (e == cudaSuccess) done_.store(true, std::memory_order_release);
    return e;
  }
};

}  // namespace vvli
