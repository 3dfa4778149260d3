// Argument checks shared by the C ABI translation units.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "m3scan.h"

namespace m3 {

// SM count and compute capability of a device do not change: asked for once
// (a query per call is a good part of a small call's time on the host).
constexpr int kMaxDevices = 64;
struct DeviceInfo {
  std::atomic<int> sms{0}, major{0};   // 0: not asked yet
};
inline DeviceInfo* device_info() {
  static DeviceInfo info[kMaxDevices];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) { cudaGetLastError(); return nullptr; }
  if (dev < 0 || dev >= kMaxDevices) return nullptr;
  DeviceInfo* d = &info[dev];
  if (d->sms.load(std::memory_order_acquire) == 0) {
    int sms = 0, major = 0;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess) {
      cudaGetLastError();
      return nullptr;
    }
    d->major.store(major, std::memory_order_relaxed);
    d->sms.store(sms, std::memory_order_release);
  }
  return d;
}

// SM count of the current device, -1 when there is none
inline int device_sms() {
  const DeviceInfo* d = device_info();
  return d ? d->sms.load(std::memory_order_relaxed) : -1;
}

inline int check_device() {
  const DeviceInfo* d = device_info();
  return d && d->major.load(std::memory_order_relaxed) == 10 ? M3_OK : M3_ERR_NO_DEVICE;
}

// Lets a kernel use `smem` bytes of dynamic shared memory, once per device and
// kernel; one value per kernel, so that calls from several threads agree.
struct OncePerDevice {
  std::atomic<int> value[kMaxDevices] = {};
};
template <auto* kern>
cudaError_t allow_smem(int smem) {
  static OncePerDevice done;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < kMaxDevices && done.value[dev].load(std::memory_order_acquire) >= smem)
    return cudaSuccess;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess && dev < kMaxDevices)
    done.value[dev].store(smem, std::memory_order_release);
  return e;
}

inline bool dtype_ok(int dt) { return dt == M3_F32 || dt == M3_BF16; }
inline int dsize(int dt) { return dt == M3_BF16 ? 2 : 4; }
inline bool aligned(const void* p, int a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
inline size_t round256(size_t x) { return (x + 255) & ~(size_t)255; }

// CTAs of a kernel that an SM holds, 0 on an error; asked for once per device.
template <auto* kern>
int resident_ctas(OncePerDevice& known, int threads, int smem) {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= kMaxDevices) { cudaGetLastError(); return 0; }
  if ((n = known.value[dev].load(std::memory_order_acquire)) > 0) return n;
  if (allow_smem<kern>(smem) != cudaSuccess ||
      cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, threads, smem) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  known.value[dev].store(n, std::memory_order_release);
  return n;
}

}  // namespace m3
