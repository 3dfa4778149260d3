// Device code shared by the selective scan's forward, backward and step.
//
// Per row b, channel d, state n:
//   de_t = softplus(dt_t + dt_bias)   (or dt_t + dt_bias)
//   h_t  = exp(de_t A) h_{t-1} + de_t u_t B_t
//   y_t  = (sum_n C_t h_t + D u_t) silu(z_t)
//
// Layout: a lane group of LN threads owns two adjacent channels; thread q of the
// group holds states Sq .. Sq+S-1 of both (S = 8 forward, 4 backward).  Steps are staged kSelSteps at a time
// through shared memory; a step past the row's length is staged with de = 0,
// which leaves the state as it is (exp(0) = 1, nothing added), so no branch on
// the length is left in the recurrence.  State products are packed pairs of
// states (fma.rn.f32x2).
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "m3_math.cuh"
#include "m3_ops.h"
#include "m3_prologue.cuh"
#include "m3_vec.cuh"

namespace m3 {

constexpr int kS = kSelSteps;

// A kernel's tiling: LN lanes per pair of channels, S states per lane and channel,
// NT threads per CTA.
template <int LN_, int S_, int NT_> struct Tiling {
  static constexpr int LN = LN_, S = S_, NT = NT_;
  static constexpr int DT = NT / LN * 2;            // channels per CTA
  static constexpr int NP = S * LN;                 // states kept per channel
  static constexpr int EPT = kS * DT / NT;          // staged elements per thread and tensor
  static constexpr int QUADS = kS * NP / 4;         // staged state quads of B (or C)
  static constexpr int QPT = (QUADS + NT - 1) / NT; // per thread
};
// Backward: four states per lane (its registers hold gates and products of four
// steps).
template <int LN> using Sel = Tiling<LN, 4, (LN >= 16 ? 256 : 128)>;
// Forward and the summaries: eight.  Every register filled from shared memory
// costs the SM a cycle of its 128 bytes per clock, however many lanes share
// the value; a lane with more states uses a step's B and C for two channels and
// its step size for eight states.
template <int LN> using SelF = Tiling<LN, 8, (LN >= 2 ? 32 * LN : 64)>;

__device__ __forceinline__ int sel_length(const int* lengths, int b, int L) {
  if (lengths == nullptr) return L;
  const int n = lengths[b];
  return n < 0 ? 0 : n > L ? L : n;
}

// softplus(x) = max(x, 0) + log(1 + t), t = e^-|x|, without the library's
// log1p and exp (about 50 instructions per element, more than a short state's
// recurrence costs): t on the MUFU unit, its argument's rounding added back to
// first order (hi + lo is |x| log2 e to twice the precision); and
// log(1 + t) = 2 artanh(s), s = t / (2 + t) <= 1/3, by its series
// s + s^3/3 + ... + s^13/13 (what is left out is below 2e-8 of it).  Relative
// error a few 1e-7 over the whole range, past torch's threshold of 20 too,
// where log(1 + t) is below half an ulp of x.
constexpr float kLog2eLo = 0x1.4ae0cp-26f;      // log2(e) - kLog2e

constexpr float kSoftplusShift = 7e-8f;
__device__ __forceinline__ float exp_neg(float ax) {   // e^-ax, ax >= 0
  const float hi = -ax * kLog2e;
  const float lo = fmaf(-ax, kLog2eLo, fmaf(-ax, kLog2e, -hi));
  const float t = ex2_approx(hi);
  // + kSoftplusShift: the units' mean error of -5e-8 (ex2, then the division)
  return ax >= 126.f ? 0.f : fmaf(t * 0x1.62e43p-1f, lo + kSoftplusShift, t);   // NaN passes
}
__device__ __forceinline__ float log1p_of(float t) {   // t in [0, 1]
  const float s = t * rcp_approx(2.f + t), q = s * s;
  float p = 1.f / 13.f;
  p = fmaf(p, q, 1.f / 11.f);
  p = fmaf(p, q, 1.f / 9.f);
  p = fmaf(p, q, 1.f / 7.f);
  p = fmaf(p, q, 1.f / 5.f);
  p = fmaf(p, q, 1.f / 3.f);
  p = fmaf(p, q, 1.f);
  return 2.f * s * p;
}
// Step size of one element (bias added, softplus or not); `slope` gets its
// derivative.
__device__ __forceinline__ float step_size(float x, int softplus) {
  if (!softplus) return x;
  return fmaxf(x, 0.f) + log1p_of(exp_neg(fabsf(x)));
}
__device__ __forceinline__ float step_size(float x, int softplus, float* slope) {
  if (!softplus) {
    *slope = 1.f;
    return x;
  }
  const float t = exp_neg(fabsf(x)), r = rcp_approx(1.f + t);
  *slope = x > 0.f ? r : t * r;
  return fmaxf(x, 0.f) + log1p_of(t);
}

// Sum over the LN lanes of a group of NV values per lane, transposed: in each
// round a lane keeps the half of the values that its lane bit names and adds
// the partner's copy, so with NV = LN lane q ends with total q in v[0], and
// with NV = c LN it holds totals q c .. q c + c - 1 in v[0 .. c-1].  NV < LN
// finishes with plain butterflies (several lanes hold the same total).  Fixed
// order.
template <int NV, int LN, int M = LN / 2>
__device__ __forceinline__ void lane_sum(float* v, int q) {
  if constexpr (M >= 1) {
    if constexpr (NV >= 2) {
      const bool up = (q & M) != 0;
#pragma unroll
      for (int i = 0; i < NV / 2; ++i) {
        const float keep = up ? v[NV / 2 + i] : v[i];
        const float send = up ? v[i] : v[NV / 2 + i];
        v[i] = keep + __shfl_xor_sync(0xffffffffu, send, M);
      }
      lane_sum<NV / 2, LN, M / 2>(v, q);
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], M);
      lane_sum<1, LN, M / 2>(v, q);
    }
  }
}

// The gates exp(de A) of two states from a2 = A log2(e).  The MUFU unit's 2^x is
// low by 2e-8 on average for x in [-1, -1e-4] (measured), a third of a last place
// below 1; a slow state multiplies hundreds of gates, and dA, which weighs them
// by age, was off by 4e-7 with one sign.  The shift of the argument by
// 2e-8 log2(e) takes the mean out; 2^shift itself rounds to 1.
constexpr float kGateShift = 2.9e-8f;
__device__ __forceinline__ float2 gate_pair(float2 de, float2 a2) {
  const float2 x = __ffma2_rn(de, a2, f2(kGateShift));
  return make_float2(ex2_approx(x.x), ex2_approx(x.y));
}

// A quad 4q .. 4q+3 of channel c in a (rows, D, N) tensor by element loads (zero
// past D or N), and in a padded (rows, D, NP) buffer.
__device__ __forceinline__ float4 load_quad_any(const float* src, size_t row, int c, int n0, int D,
                                                int N) {
  float v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    v[j] = (src != nullptr && c < D && n0 + j < N) ? src[(row * D + c) * N + n0 + j] : 0.f;
  return make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store_quad_any(float4 x, float* dst, size_t row, int c, int n0,
                                               int D, int N) {
  const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (c < D && n0 + j < N) dst[(row * D + c) * N + n0 + j] = v[j];
}
__device__ __forceinline__ float4 load_quad_pad(const float* src, size_t row, int c, int n0, int D,
                                                int NP) {
  return c < D ? *reinterpret_cast<const float4*>(src + (row * D + c) * NP + n0)
               : make_float4(0.f, 0.f, 0.f, 0.f);
}
__device__ __forceinline__ void store_quad_pad(float4 v, float* dst, size_t row, int c, int n0,
                                               int D, int NP) {
  if (c < D) *reinterpret_cast<float4*>(dst + (row * D + c) * NP + n0) = v;
}
__device__ __forceinline__ void set_pairs(float2* h, float4 v) {
  h[0] = make_float2(v.x, v.y);
  h[1] = make_float2(v.z, v.w);
}
__device__ __forceinline__ float4 quad_of(const float2* h) {
  return make_float4(h[0].x, h[0].y, h[1].x, h[1].y);
}
// A to powers of 2.  A below -1e38 (-infinity among them) counts as that: its gate
// is 0 at any step size, but 1 where the step size is 0 (a step past the length).
__device__ __forceinline__ float power_of(float a) {
  const float v = a * kLog2e;
  return v < -1e38f ? -1e38f : v;   // NaN stays
}
__device__ __forceinline__ float4 powers_of(float4 a) {
  return make_float4(power_of(a.x), power_of(a.y), power_of(a.z), power_of(a.w));
}
// A run's gate 2^e on a state: a zero stays, even where growth over the whole run
// (A > 0) overflows.
__device__ __forceinline__ float carry_over(float e, float h, float sum) {
  return h == 0.f ? sum : fmaf(ex2_approx(e), h, sum);
}

// ------------------------------------------------------------- staged rows
// Element e of a thread in a (kS, DT) tile: VW consecutive channels at a time.
template <typename T, typename G> struct TileMap {
  static constexpr int VMAX = 16 / (int)sizeof(T);
  static constexpr int VW = G::EPT < VMAX ? G::EPT : VMAX;   // channels per load
  static constexpr int NVEC = G::EPT / VW;
  static constexpr int PER_ROW = G::DT / VW;
  static __device__ __forceinline__ int row(int i) {
    return ((int)threadIdx.x + i * G::NT) / PER_ROW;
  }
  static __device__ __forceinline__ int col(int i) {
    return ((int)threadIdx.x + i * G::NT) % PER_ROW * VW;
  }
};

// Where the pair of channels (2 p, 2 p + 1) of a staged row stands, in pairs of 16
// bytes: a thread stages VW neighbouring channels, so without a permutation the
// threads of a warp would meet in VW / 4 of the banks.
template <typename M>
__device__ __forceinline__ int pair_at(int p) {
  constexpr int UPT = M::VW >= 2 ? M::VW / 2 : 1;
  return p ^ ((p >> 3) & (UPT - 1));
}

// A thread's own copy of what it will stage, filled ahead of use: 4, 8 or 16
// bytes at a time by cp.async, so that loads are in flight over a whole group of
// steps without holding registers.  Only the thread that copied reads it back
// (after copies_wait), so no barrier is needed.
__device__ __forceinline__ void copies_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}
template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst, const void* src, bool in) {
  const unsigned d = (unsigned)__cvta_generic_to_shared(dst);
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(d), "l"(src), "n"(BYTES),
               "r"(in ? BYTES : 0) : "memory");   // not in range: zeros
}

// The thread's elements of rows [t0, t0 + kS) of a (L, ld) tensor whose first row
// is base into its slots (slot[i] of thread x at slots[i * NT + x]); rows at or
// past n and channels past D become zero.
template <typename T, typename G>
__device__ __forceinline__ void fetch_tile(Pack<T, TileMap<T, G>::VW>* slots, const T* base,
                                           long long ld, int t0, int n, int c0, int D, bool vec) {
  using M = TileMap<T, G>;
  constexpr int BYTES = M::VW * (int)sizeof(T);
#pragma unroll
  for (int i = 0; i < M::NVEC; ++i) {
    const int t = t0 + M::row(i), c = c0 + M::col(i);
    const bool in = t < n && c < D;
    const T* p = base + (in ? (size_t)t * ld + c : 0);
    Pack<T, M::VW>* dst = slots + i * G::NT + threadIdx.x;
    if (BYTES >= 4 && vec) {   // D is a multiple of VW
      copy_async<(BYTES >= 4 ? BYTES : 4)>(dst, p, in);
    } else {
      Pack<T, M::VW> v = zero_pack<T, M::VW>();
      if (in)
#pragma unroll
        for (int j = 0; j < M::VW; ++j)
          if (c + j < D) v.load_one(j, p);
      *dst = v;
    }
  }
}
template <typename T, typename G>
__device__ __forceinline__ void store_tile(const Pack<T, TileMap<T, G>::VW>& v, int i, T* base,
                                           long long ld, int t0, int L, int c0, int D, bool vec) {
  using M = TileMap<T, G>;
  const int t = t0 + M::row(i), c = c0 + M::col(i);
  if (t < L && c < D) {
    T* p = base + (size_t)t * ld + c;
    if (vec) st_pack<T, M::VW>(p, v);
    else
#pragma unroll
      for (int j = 0; j < M::VW; ++j)
        if (c + j < D) v.store_one(j, p);
  }
}

// The thread's state quads of rows [t0, t0 + kS) of B or C into its slots.
template <typename T, typename G>
__device__ __forceinline__ void fetch_quads(Pack<T, 4>* slots, const T* base, long long ld, int t0,
                                            int n, int N, bool vec) {
#pragma unroll
  for (int i = 0; i < G::QPT; ++i) {
    const int e = (int)threadIdx.x + i * G::NT;
    const int t = t0 + e / (G::NP / 4), k = e % (G::NP / 4) * 4;
    const bool in = e < G::QUADS && t < n && k < N;
    const T* p = base + (in ? (size_t)t * ld + k : 0);
    Pack<T, 4>* dst = slots + i * G::NT + threadIdx.x;
    if (vec) {                 // N is a multiple of 4
      copy_async<4 * (int)sizeof(T)>(dst, p, in);
    } else {
      Pack<T, 4> v = zero_pack<T, 4>();
      if (in)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (k + j < N) v.load_one(j, p);
      *dst = v;
    }
  }
}

}  // namespace m3
