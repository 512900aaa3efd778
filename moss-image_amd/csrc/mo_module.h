// What the launchers of one code object share: its kernels by name, loaded once for each device.
#pragma once
#include <hip/hip_runtime_api.h>

#include <atomic>
#include <map>
#include <mutex>
#include <string>

#include "../../include/moss_offload.h"

namespace mo {

int set_error(int code, const std::string& msg);
int set_hip_error(int e, const char* what);

class Kernels {
 public:
  static constexpr int kIds = 128, kDevices = 16;

  explicit Kernels(const unsigned char* code) : code_(code) {}

  // The kernel `name()` on the current device; `id` below kIds is the same name every time. Found once, without a lock.
  template <class Name>
  int get(int id, Name&& name, hipFunction_t* out) {
    int device = 0;
    hipError_t e = hipGetDevice(&device);
    if (e != hipSuccess) return set_hip_error((int)e, "hipGetDevice");
    std::atomic<hipFunction_t>* known = device < kDevices ? &known_[device][id] : nullptr;
    if (known && (*out = known->load(std::memory_order_acquire))) return 0;
    std::lock_guard<std::mutex> lock(mu_);
    auto module = modules_.find(device);
    if (module == modules_.end()) {
      hipModule_t m = nullptr;
      if ((e = hipModuleLoadData(&m, code_)) != hipSuccess) return set_hip_error((int)e, "hipModuleLoadData");
      module = modules_.emplace(device, m).first;
    }
    hipFunction_t f = nullptr;
    if ((e = hipModuleGetFunction(&f, module->second, std::string(name()).c_str())) != hipSuccess)
      return set_hip_error((int)e, "hipModuleGetFunction");
    if (known) known->store(f, std::memory_order_release);
    *out = f;
    return 0;
  }

 private:
  const unsigned char* code_;
  std::mutex mu_;
  std::map<int, hipModule_t> modules_;
  std::atomic<hipFunction_t> known_[kDevices][kIds] = {};
};

inline int launch(hipFunction_t f, uint32_t gx, uint32_t gy, uint32_t gz, uint32_t threads, uint64_t stream, void** params,
                  const char* what) {
  const hipError_t e =
      hipModuleLaunchKernel(f, gx, gy, gz, threads, 1, 1, 0, (hipStream_t)stream, params, nullptr);
  return e == hipSuccess ? 0 : set_hip_error((int)e, what);
}

// No exception crosses the C boundary (a failed allocation in a map or a message is what could).
template <class F>
int guarded(F&& body) {
  try {
    return body();
  } catch (...) {
    return set_error(MO_E_HOST_OOM, "no host memory");  // short: needs no allocation itself
  }
}

}  // namespace mo
