// Shared pieces of the gated linear recurrence's kernels.
//
//   r = sigmoid(rg), i = sigmoid(ig), l = -c softplus(decay) r  (<= 0)
//   a = e^l, m = sqrt(1 - a^2),   h_t = a_t h_{t-1} + m_t i_t x_t
//
// A decay near 1 is what these layers are made of, and an error of a counts
// 1 / (1 - a) times in the state, so a and 1 - a^2 both come from p = e^l - 1
// computed to its own precision: a = 1 + p, 1 - a^2 = -p (2 + p).  e^l - 1 is
// 2^n e^f - 1 with l = n ln 2 + f (Cody and Waite's two-part ln 2), |f| <= 0.35,
// and the Taylor sum of e^f - 1 to f^7 (next term below 2e-8 of f).  On the MUFU
// unit's ex2 instead, whose results are low by 2e-8 on average, a state would be
// low by that times 1 / (1 - a): 2e-5 at a = 0.999.
//
// All pairs below are two channels in one packed register pair.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "m3_math.cuh"
#include "m3_vec.cuh"

namespace m3 {

constexpr int kGatedSteps = 8;        // steps per thread at a time = checkpoint interval
constexpr int kGatedTile = 64;        // channels per CTA: two per lane

__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 sub2(float2 a, float2 b) { return __ffma2_rn(b, f2(-1.f), a); }

__device__ __forceinline__ float max_nan(float a, float b) {   // NaN stays NaN
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float rsqrt_approx(float x) {
  float y;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float2 sigmoid2(float2 x) {
  return make_float2(sigmoid_f(x.x), sigmoid_f(x.y));
}

// log(1 + e^x), of the decay parameter: once per thread
__device__ __forceinline__ float softplus_f(float x) {
  return x > 20.f ? x : log1pf(expf(x));
}

// a = e^l and p = e^l - 1 for l <= 0 (l below -87: as -87, where a is 2e-38)
__device__ __forceinline__ void decay2(float2 l, float2& a, float2& p) {
  constexpr float kLn2Hi = 0x1.62e4p-1f;          // ln 2 to 16 bits: n times it is exact
  constexpr float kLn2Lo = 0x1.7f7d1cp-20f;       // ln 2 - kLn2Hi
  l = make_float2(max_nan(l.x, -87.f), max_nan(l.y, -87.f));
  const float2 j = fma2(l, f2(kLog2e), f2(kMagic));
  const float2 n = add2(j, f2(-kMagic));
  float2 f = fma2(n, f2(-kLn2Hi), l);
  f = fma2(n, f2(-kLn2Lo), f);
  float2 q = fma2(f, f2(1.f / 5040.f), f2(1.f / 720.f));
  q = fma2(q, f, f2(1.f / 120.f));
  q = fma2(q, f, f2(1.f / 24.f));
  q = fma2(q, f, f2(1.f / 6.f));
  q = fma2(q, f, f2(0.5f));
  const float2 e = fma2(mul2(f, f), q, f);        // e^f - 1
  // 2^n: the low bits of j hold n
  const float2 s = make_float2(
      __uint_as_float((__float_as_uint(j.x) << 23) + 0x3f800000u),
      __uint_as_float((__float_as_uint(j.y) << 23) + 0x3f800000u));
  a = fma2(s, e, s);
  p = fma2(s, e, add2(s, f2(-1.f)));
}

// m = sqrt(-p (2 + p)) and 1 / m (finite where m is 0)
__device__ __forceinline__ void root2(float2 p, float2& m, float2& inv) {
  const float2 v = mul2(p, fma2(p, f2(-1.f), f2(-2.f)));
  inv = make_float2(rsqrt_approx(fmaxf(v.x, 1e-37f)), rsqrt_approx(fmaxf(v.y, 1e-37f)));
  m = mul2(v, inv);
}

// v_out = P v_in + V over a run of steps, per channel
struct Run {
  float2 P, V;
};
__device__ __forceinline__ void then(Run& first, const Run& next) {   // first, then next
  first.V = fma2(next.P, first.V, next.V);
  first.P = mul2(next.P, first.P);
}

// ------------------------------------------------------------------ staging
// A warp's rows of NA arrays, kGatedSteps steps of kGatedTile channels each, as
// they lie in memory.  Each warp copies and reads its own rows only.
template <typename T, int NA>
struct Stage {
  static constexpr int kRow = kGatedTile * (int)sizeof(T);         // bytes
  static constexpr int kBytes = NA * kGatedSteps * kRow;           // per warp
  const T* src[NA]; long long ld[NA];

  // rows t0 .. of row `base` (b L), those below `n`; channels c0 .. below D
  __device__ __forceinline__ void issue(char* buf, long long base, int t0, int n, int c0, int D,
                                        bool vec) const {
    const int lane = threadIdx.x;
    if (vec) {
      constexpr int V = 16 / (int)sizeof(T), PR = kGatedTile / V;
#pragma unroll
      for (int k = 0; k < NA; ++k)
#pragma unroll
        for (int i = 0; i < kGatedSteps * PR / 32; ++i) {
          const int at = i * 32 + lane, t = t0 + at / PR, c = c0 + at % PR * V;
          const bool ok = t < n && c < D;
          const T* g = src[k] + (ok ? (size_t)(base + t) * ld[k] + c : 0);
          const unsigned s = (unsigned)__cvta_generic_to_shared(buf + k * kGatedSteps * kRow +
                                                                at * 16);
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(s), "l"(g),
                       "r"(ok ? 16 : 0)
                       : "memory");
        }
      asm volatile("cp.async.commit_group;" ::: "memory");
    } else {
      const int c = c0 + 2 * lane;
#pragma unroll
      for (int k = 0; k < NA; ++k)
        for (int i = 0; i < kGatedSteps; ++i) {
          const bool ok = t0 + i < n;
          const T* g = src[k] + (ok ? (size_t)(base + t0 + i) * ld[k] + c : 0);
          T* s = reinterpret_cast<T*>(buf + (k * kGatedSteps + i) * kRow) + 2 * lane;
          s[0] = ok && c < D ? g[0] : T(0.f);
          s[1] = ok && c + 1 < D ? g[1] : T(0.f);
        }
    }
  }
  static __device__ __forceinline__ void wait() {
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();
  }
  // the lane's pair of step i of array k
  static __device__ __forceinline__ float2 get(const char* buf, int k, int i) {
    const Pack<T, 2> v = ld_pack<T, 2>(reinterpret_cast<const T*>(buf + (k * kGatedSteps + i) * kRow) +
                                       2 * threadIdx.x);
    return make_float2(v.get(0), v.get(1));
  }
};

// A lane's pair of channels in a (.., D) array, element by element where a pair
// may be cut or is not aligned.
template <typename T>
__device__ __forceinline__ void store_pair(T* p, float2 v, int left, bool vec) {
  if (vec) {
    if (left > 0) {
      Pack<T, 2> o;
      o.put(0, v.x);
      o.put(1, v.y);
      st_pack<T, 2>(p, o);
    }
  } else {
    if (left > 0) p[0] = Elem<T>::put(v.x);
    if (left > 1) p[1] = Elem<T>::put(v.y);
  }
}
__device__ __forceinline__ float2 load_pair(const float* p, int left) {
  return make_float2(left > 0 ? p[0] : 0.f, left > 1 ? p[1] : 0.f);
}

// ------------------------------------------------------------------ joins
// The CTA's warps and, for S > 1, the cluster's CTAs hold consecutive runs of
// steps (`order`: this warp's place in the CTA's order, `rank` this CTA's in the
// cluster's).  Every thread folds the runs ahead of its own onto the value
// `carry` before the first, and carry moves behind the last.  Two buffers in turn:
// one CTA barrier (and one cluster barrier) per call.
struct Joint {
  float4 warp[2][8][32];
  float4 cta[2][8][32];
};

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}

__device__ __forceinline__ float2 join(Joint& j, int flip, const Run& mine, int order, int warps,
                                       int rank, int S, float2& carry) {
  const int lane = threadIdx.x;
  j.warp[flip][order][lane] = make_float4(mine.P.x, mine.P.y, mine.V.x, mine.V.y);
  __syncthreads();
  Run all{f2(1.f), f2(0.f)}, ahead = all;
  for (int w = 0; w < warps; ++w) {
    if (w == order) ahead = all;
    const float4 v = j.warp[flip][w][lane];
    then(all, Run{make_float2(v.x, v.y), make_float2(v.z, v.w)});
  }
  float2 start = carry;
  if (S > 1) {
    for (int peer = threadIdx.y; peer < S; peer += warps) {
      unsigned a = (unsigned)__cvta_generic_to_shared(&j.cta[flip][rank][lane]), to;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(a), "r"(peer));
      asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(all.P.x),
                   "f"(all.P.y), "f"(all.V.x), "f"(all.V.y)
                   : "memory");
    }
    cluster_sync();
    float2 c = carry;
    for (int k = 0; k < S; ++k) {
      if (k == rank) start = c;
      const float4 v = j.cta[flip][k][lane];
      c = fma2(make_float2(v.x, v.y), c, make_float2(v.z, v.w));
    }
    carry = c;
  } else {
    carry = fma2(all.P, carry, all.V);
  }
  return fma2(ahead.P, start, ahead.V);
}

}  // namespace m3
