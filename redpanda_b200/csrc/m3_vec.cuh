// Vector loads and stores of float or bf16 elements as fp32 values.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace m3 {

template <typename T> struct Elem;
template <> struct Elem<float> {
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
template <> struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};

// V consecutive elements held as loaded (V * sizeof(T) = 2, 4, 8, 16 or 32
// bytes; the address must be aligned to min(that, 16)).
template <typename T, int V>
struct alignas(V * sizeof(T) < 16 ? V * sizeof(T) : 16) Pack {
  T v[V];
  __device__ __forceinline__ float get(int i) const { return Elem<T>::get(v[i]); }
  __device__ __forceinline__ void put(int i, float x) { v[i] = Elem<T>::put(x); }
};

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> ld_pack(const T* p) {
  return *reinterpret_cast<const Pack<T, V>*>(p);
}

template <typename T, int V>
__device__ __forceinline__ void st_pack(T* p, const Pack<T, V>& x) {
  *reinterpret_cast<Pack<T, V>*>(p) = x;
}

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> zero_pack() {
  Pack<T, V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = Elem<T>::put(0.f);
  return r;
}

// silu and its derivative in fp32: s = 1 / (1 + e^-x), silu = x s,
// silu' = s (1 + x (1 - s)).  __expf and the fast division are within a few
// fp32 ulp, below the rounding of a bf16 result and near that of an fp32 one;
// e^-x overflows to infinity for x < -88, where s is 0 as it should be.
__device__ __forceinline__ float sigmoid_f(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }
__device__ __forceinline__ float silu_f(float x) { return x * sigmoid_f(x); }
__device__ __forceinline__ float dsilu_f(float x, float s) { return s * (1.f + x * (1.f - s)); }

}  // namespace m3
