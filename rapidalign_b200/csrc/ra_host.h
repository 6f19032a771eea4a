// ra_host.h -- host helpers shared by the translation units of the library.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstddef>
#include <cstdint>

#include "../../include/rapidalign_b200.h"

namespace ra {

extern std::atomic<unsigned long long> g_launches;  // kernels launched (ra_capi.cu)

inline size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }
inline int sm_count() {
  int dev = 0, sms = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms > 0 ? sms : 1;
}
// Something that is done once for each device (a kernel's attributes).  Doing
// it twice, from two threads at once, does no harm.
struct OncePerDevice {
  std::atomic<unsigned long long> done{0};  // devices 0 .. 63
  template <class F>
  bool operator()(F f) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return false;
    if (dev < 64 && (done.load() >> dev & 1)) return true;
    if (!f()) return false;
    if (dev < 64) done.fetch_or(1ull << dev);
    return true;
  }
};
inline int launched() {
  ++g_launches;
  return cudaGetLastError() == cudaSuccess ? RA_OK : RA_ERR_CUDA;
}

}  // namespace ra
