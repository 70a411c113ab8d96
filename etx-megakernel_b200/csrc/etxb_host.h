// What the library's translation units share on the host: the text of the last failure, and the device of a call.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

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
