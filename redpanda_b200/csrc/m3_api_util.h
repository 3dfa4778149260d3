// Argument checks shared by the C ABI translation units.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "m3scan.h"

namespace m3 {

// SM count of the current device, -1 when there is none
inline int device_sms() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) { cudaGetLastError(); return -1; }
  int sms = 0;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
    cudaGetLastError();
    return -1;
  }
  return sms;
}

inline int check_device() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) { cudaGetLastError(); return M3_ERR_NO_DEVICE; }
  int major = 0;
  if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess) {
    cudaGetLastError();
    return M3_ERR_NO_DEVICE;
  }
  return major == 10 ? M3_OK : M3_ERR_NO_DEVICE;
}

inline bool dtype_ok(int dt) { return dt == M3_F32 || dt == M3_BF16; }
inline int dsize(int dt) { return dt == M3_BF16 ? 2 : 4; }
inline bool aligned(const void* p, int a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
inline size_t round256(size_t x) { return (x + 255) & ~(size_t)255; }

}  // namespace m3
