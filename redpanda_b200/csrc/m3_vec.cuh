// Vector loads and stores of float or bf16 elements as fp32 values.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "m3_math.cuh"

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
// bytes; the address must be aligned to min(that, 16)).  bf16 pairs stay in
// 32-bit words until they are read: an array of 16-bit values would be taken
// apart where it is loaded, and a load made ahead of its use would be waited for
// there (the selective scan's bf16 forward ran at half the speed that way).
// Elements are put in ascending order.
template <typename T, int V> struct Pack;

template <int V>
struct alignas(V * 4 < 16 ? V * 4 : 16) Pack<float, V> {
  float v[V];
  __device__ __forceinline__ float get(int i) const { return v[i]; }
  __device__ __forceinline__ void put(int i, float x) { v[i] = x; }
  __device__ __forceinline__ void load_one(int i, const float* p) { v[i] = p[i]; }
  __device__ __forceinline__ void store_one(int i, float* p) const { p[i] = v[i]; }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = 0.f;
  }
};

template <int V>
struct alignas(V * 2 < 16 ? V * 2 : 16) Pack<__nv_bfloat16, V> {
  unsigned w[V / 2];
  __device__ __forceinline__ float get(int i) const {
    return __uint_as_float((i & 1) ? (w[i / 2] & 0xffff0000u) : (w[i / 2] << 16));
  }
  __device__ __forceinline__ void put(int i, float x) {
    const unsigned b = __bfloat16_as_ushort(__float2bfloat16_rn(x));
    w[i / 2] = (i & 1) ? (w[i / 2] | b << 16) : b;
  }
  __device__ __forceinline__ void load_one(int i, const __nv_bfloat16* p) {
    const unsigned b = reinterpret_cast<const unsigned short*>(p)[i];
    w[i / 2] = (i & 1) ? ((w[i / 2] & 0xffffu) | b << 16) : ((w[i / 2] & 0xffff0000u) | b);
  }
  __device__ __forceinline__ void store_one(int i, __nv_bfloat16* p) const {
    reinterpret_cast<unsigned short*>(p)[i] =
        (unsigned short)((i & 1) ? w[i / 2] >> 16 : w[i / 2] & 0xffffu);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) w[i] = 0u;
  }
};

template <>
struct Pack<__nv_bfloat16, 1> {
  unsigned short w;
  __device__ __forceinline__ float get(int) const { return __uint_as_float((unsigned)w << 16); }
  __device__ __forceinline__ void put(int, float x) {
    w = __bfloat16_as_ushort(__float2bfloat16_rn(x));
  }
  __device__ __forceinline__ void load_one(int, const __nv_bfloat16* p) {
    w = *reinterpret_cast<const unsigned short*>(p);
  }
  __device__ __forceinline__ void store_one(int, __nv_bfloat16* p) const {
    *reinterpret_cast<unsigned short*>(p) = w;
  }
  __device__ __forceinline__ void zero() { w = 0; }
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
  r.zero();
  return r;
}

// silu and its derivative in fp32: s = 1 / (1 + e^-x), silu = x s,
// silu' = s + x s (1 - s), on the MUFU unit.  The exponent x log2(e) is rounded
// once, so the relative error is up to (1.3 |x| + 10) 2^-24: a few fp32 ulp, and
// below the rounding of a bf16 result, where the gate matters, 2e-6 of a gate of
// 4e-8 at x = -20.  1 + e^-x past 2^126 has the reciprocal 0, so below x = -87.3
// both are 0 (silu itself is below 1.1e-36 there).
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float sigmoid_f(float x) {
  return rcp_approx(1.f + ex2_approx(x * -kLog2e));
}
__device__ __forceinline__ float silu_f(float x) { return x * sigmoid_f(x); }
__device__ __forceinline__ float dsilu_f(float x, float s) {
  const float xs = x * s;
  return fmaf(-xs, s, xs) + s;
}

}  // namespace m3
