// Shared pieces of the norm kernels: a row's elements in registers, sums over a
// row, and the instantiation of a row length (m3_norm.cu has the reasons).
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "m3_api_util.h"
#include "m3_vec.cuh"

namespace m3 {
namespace {

// Sum of N values over the threads of a row, every thread gets the totals: a
// warp (WARP), or the CTA, through one of two buffers in turn (`flip`), so that
// one barrier per sum is enough.
template <bool WARP, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*red)[64], int& flip) {
#pragma unroll
  for (int m = 16; m > 0; m >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], m);
  if constexpr (!WARP) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, W = blockDim.x >> 5;
    float* r = red[flip];
    flip ^= 1;
    if (lane == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) r[i * 32 + warp] = v[i];
    __syncthreads();
    if (W <= 4) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float s = r[i * 32];
        for (int w = 1; w < W; ++w) s += r[i * 32 + w];
        v[i] = s;
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float s = lane < W ? r[i * 32 + lane] : 0.f;
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
        v[i] = s;
      }
    }
  }
}

// A thread's elements: VEC consecutive columns from (i * tpr + t) * VEC.
template <typename T, int VEC, int NV>
struct Row {
  Pack<T, VEC> p[NV];
  __device__ __forceinline__ void load(const T* row, int d, int t, int tpr) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * tpr + t) * VEC;
      p[i] = c < d ? ld_pack<T, VEC>(row + c) : zero_pack<T, VEC>();
    }
  }
  __device__ __forceinline__ float get(int k) const { return p[k / VEC].get(k % VEC); }
};

template <int VEC, int NV>
__device__ __forceinline__ void load_f32(float (&w)[VEC * NV], const float* src, int d, int t,
                                         int tpr) {
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int c = (i * tpr + t) * VEC + j;
      w[i * VEC + j] = (src != nullptr && c < d) ? src[c] : 0.f;
    }
}

// Threads of a row's CTA (0: a warp per row).
inline int norm_threads(int d) {
  if (d <= 256) return 0;
  const int per = d <= 8192 ? 8 : 32;
  return (d + 32 * per - 1) / (32 * per) * 32;
}
// CTAs per SM of the persistent grids: 768 threads, as many as 80 registers per
// thread allow (one CTA where a thread holds 32 elements or has 64 registers).
inline int norm_per_sm(int d, int nt) { return d > 8192 || nt > 768 ? 1 : 768 / nt; }

// vec: widest vector (8 when both sides are bf16, else 4) that the row starts
// and lengths allow, else single elements.
inline int norm_vec(int d, int dtype_x, int dtype_y, bool ok8, bool ok4) {
  if (dtype_x == M3_BF16 && dtype_y == M3_BF16 && ok8 && d % 8 == 0) return 8;
  return ok4 && d % 4 == 0 ? 4 : 1;
}

// The instantiation of a row length: f<VEC, NV, WARP, MAXT, MINB>(threads).  Vectors of 8
// where F has kWide, in warps of 2 where it has kEven.  Here a CTA's rows:
template <int E, typename F>
cudaError_t norm_size(int vec, int nt, F&& f) {
  auto with = [&](auto v) -> cudaError_t {
    constexpr int VEC = decltype(v)::value, NV = E / VEC;
    if constexpr (E == 8) {
      if (nt <= 768) return f.template operator()<VEC, NV, false, 768, 1>(nt);
    } else {
      if (nt <= 512) return f.template operator()<VEC, NV, false, 512, 1>(nt);
    }
    return f.template operator()<VEC, NV, false, 1024, 1>(nt);
  };
  if constexpr (std::decay_t<F>::kWide)
    if (vec == 8) return with(std::integral_constant<int, 8>());
  return vec == 4 ? with(std::integral_constant<int, 4>())
                  : with(std::integral_constant<int, 1>());
}
// Rows a warp holds at E elements per lane.
template <int E, typename F>
cudaError_t norm_warp(int vec, F&& f) {
  constexpr int MINB = E <= 8 ? 6 : E <= 16 ? 5 : 4;
  if constexpr (std::decay_t<F>::kWide)
    if (vec == 8) return f.template operator()<8, E / 8, true, 128, MINB>(128);
  if constexpr (std::decay_t<F>::kEven)
    if (vec == 2) return f.template operator()<2, E / 2, true, 128, MINB>(128);
  return vec == 4 ? f.template operator()<4, E / 4, true, 128, MINB>(128)
                  : f.template operator()<1, E, true, 128, MINB>(128);
}
template <typename F>
cudaError_t norm_dispatch(int d, int vec, F&& f) {
  const int nt = norm_threads(d);
  if (nt == 0) return norm_warp<8>(vec, f);
  if constexpr (std::decay_t<F>::kWarpRows) {
    if (d > 256 && d <= 512) return norm_warp<16>(vec, f);
    if (d > 512 && d <= 768) return norm_warp<24>(vec, f);
    if (d > 768 && d <= 1024) return norm_warp<32>(vec, f);
  }
  return d <= 8192 ? norm_size<8>(vec, nt, f) : norm_size<32>(vec, nt, f);
}

}  // namespace
}  // namespace m3
