// What the library's translation units share on the host: the text of the last failure, and the device of a call.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include <atomic>

#include "../../include/etxb200.h"

// Records the text etxb_last_error() returns (defined in etxb.cu) and passes the code on.  Throws nothing.
__attribute__((visibility("hidden"))) int32_t etxb_host_fail(int32_t code, const char* msg) noexcept;

#define ETXB_HOST_CU(call)                                                                      \
  do {                                                                                          \
    cudaError_t e_ = (call);                                                                    \
    if (e_ != cudaSuccess) {                                                                    \
      char m_[256];                                                                             \
      snprintf(m_, sizeof m_, "%s: %s", #call, cudaGetErrorString(e_));                         \
      return etxb_host_fail(ETXB_E_CUDA, m_);                                                   \
    }                                                                                           \
  } while (0)

// The number of a device's processors (asked once).
inline cudaError_t etxb_host_sms(int device, int* sms) {
  static std::atomic<int> known[64];
  int n = known[device].load(std::memory_order_relaxed);
  if (n == 0) {
    const cudaError_t e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device);
    if (e != cudaSuccess) return e;
    known[device].store(n, std::memory_order_relaxed);
  }
  *sms = n;
  return cudaSuccess;
}
// Lets a kernel have `bytes` of dynamic shared memory on the current device; `done`: 64 flags of the kernel's own, one a device (asked for once).
inline cudaError_t etxb_host_smem(const void* kernel, int bytes, int device, std::atomic<char>* done) {
  if (done[device].load(std::memory_order_relaxed)) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done[device].store(1, std::memory_order_relaxed);
  return e;
}

// The device of a call is current while the call runs; the caller's own is current again behind it.
struct EtxbDeviceScope {
  int prev = -1;
  cudaError_t err = cudaSuccess;
  explicit EtxbDeviceScope(int device) {
    int now = -1;
    err = cudaGetDevice(&now);
    if (err == cudaSuccess && now != device) {
      err = cudaSetDevice(device);
      if (err == cudaSuccess) prev = now;
    }
  }
  ~EtxbDeviceScope() { if (prev >= 0) cudaSetDevice(prev); }
  EtxbDeviceScope(const EtxbDeviceScope&) = delete;
  EtxbDeviceScope& operator=(const EtxbDeviceScope&) = delete;
};
