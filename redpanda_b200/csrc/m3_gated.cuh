// Shared pieces of the gated linear recurrence's kernels.
//
//   r = sigmoid(rg), i = sigmoid(ig), l = -c softplus(decay) r  (<= 0)
//   a = e^l, m = sqrt(1 - a^2),   h_t = a_t h_{t-1} + m_t i_t x_t
//
// A decay near 1 is what these layers are made of, and an error of a counts
// 1 / (1 - a) times in the state, so a and 1 - a^2 both come from p = e^l - 1
// computed to its own precision: a = 1 + p, 1 - a^2 = -p (2 + p).  e^l - 1 is
// 2^n e^f - 1 with l = n ln 2 + f, |f| <= 0.35, and e^f - 1 = f + f^2 q(f), q of
// degree 4: this project's own least-squares fit on Chebyshev nodes, weighted for
// e^f - 1's relative error, which is 1.6e-8 at most.  On the MUFU
// unit's ex2 instead, whose results are low by 2e-8 on average, a state would be
// low by that times 1 / (1 - a): 2e-5 at a = 0.999.
//
// All pairs below are two channels in one packed register pair: with scalar
// instructions instead the forward took 82 against 75 us (256 x 64 x 2048 bf16).
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "m3_bulk.cuh"
#include "m3_math.cuh"
#include "m3_vec.cuh"

namespace m3 {

constexpr int kGatedCkpt = 4;         // steps between the backward's checkpoints
// Steps of a thread at a time.  Forward 4 means as many joins again (prompt of 16384 x
// 1024 bf16: 56 against 50 us); backward 8 holds six values for each in registers and
// spills (256 x 64 x 2048 bf16: 161 against 139 us before other changes).
constexpr int kGatedFwdSteps = 8, kGatedBwdSteps = 4;
constexpr int kGatedWarps = 8;                          // of a CTA, at most

__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }

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
__device__ __forceinline__ float2 sigmoid2(float2 x) {   // sigmoid_f, packed
  const float2 t = mul2(x, f2(-kLog2e));
  const float2 u = add2(make_float2(ex2_approx(t.x), ex2_approx(t.y)), f2(1.f));
  return make_float2(rcp_approx(u.x), rcp_approx(u.y));
}

// log(1 + e^x), of the decay parameter: once per thread
__device__ __forceinline__ float softplus_f(float x) {
  return x > 20.f ? x : log1pf(expf(x));
}

// a = e^l and p = e^l - 1 for l <= 0; a is 0 from l = -87 down, where e^l is 2e-38 (a
// gradient holds l a, which would grow with l otherwise).  NEAR: l >= -kNear, where n
// is 0; the same bits with half the instructions.
constexpr float kNear = 0.34f;        // below ln(2) / 2
template <bool NEAR>
__device__ __forceinline__ void decay2(float2 l, float2& a, float2& p) {
  constexpr float kLn2 = 0x1.62e430p-1f;          // off by 2e-9, which n times is a's error
  float2 f = l, j;
  if (!NEAR) {
    l = make_float2(max_nan(l.x, -87.f), max_nan(l.y, -87.f));
    j = fma2(l, f2(kLog2e), f2(kMagic));
    f = fma2(add2(j, f2(-kMagic)), f2(-kLn2), l);
  }
  float2 q = fma2(f, f2(0x1.6d9956p-10f), f2(0x1.122838p-7f));
  q = fma2(q, f, f2(0x1.555486p-5f));
  q = fma2(q, f, f2(0x1.5554b0p-3f));
  q = fma2(q, f, f2(0.5f));
  const float2 e = fma2(mul2(f, f), q, f);        // e^f - 1
  if (NEAR) {
    a = add2(e, f2(1.f));
    p = e;
  } else {
    // 2^n: the low bits of j hold n
    const float2 s = make_float2(
        __uint_as_float((__float_as_uint(j.x) << 23) + 0x3f800000u),
        __uint_as_float((__float_as_uint(j.y) << 23) + 0x3f800000u));
    a = fma2(s, e, s);
    if (l.x == -87.f) a.x = 0.f;
    if (l.y == -87.f) a.y = 0.f;
    p = fma2(s, e, add2(s, f2(-1.f)));
  }
}

// m = sqrt(-p (2 + p)) and 1 / m, finite where m is 0 (1e-37 is far below what m
// can be but for that: 2 |l| is 1e-37 where the gate is 1e-38)
__device__ __forceinline__ void root2(float2 p, float2& m, float2& inv) {
  const float2 v = mul2(p, fma2(p, f2(-1.f), f2(-2.f)));
  const float2 w = add2(v, f2(1e-37f));
  inv = make_float2(rsqrt_approx(w.x), rsqrt_approx(w.y));
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

// ------------------------------------------------------------------ layout
// LC lanes hold a run of TS steps, two channels each; a warp holds 32 / LC
// consecutive runs of a tile of 2 LC channels.
template <int LC, int TS> struct Lanes {
  static constexpr int kSub = 32 / LC, kTile = 2 * LC, kSteps = TS * kSub;
};

// How rows are copied, by what their starts and lengths allow: 16 bytes at a time,
// words (fp32, and bf16 rows of whole words), or words that bf16 rows start in the
// middle of.  All asynchronous: with plain loads a row that is not aligned to 16 bytes
// is waited for where it is asked for (2 x 16001 x 1281 fp32: 447 against 165 us
// forward, 832 against 333 backward; 256 x 64 x 2047 bf16, half words: 224 against 163
// and 520 against 322; 2046, words: 224 against 75 and 511 against 146).
enum Copy { kHalfWords = 0, kWords = 1, kVectors = 2 };

// A warp's rows of NA arrays: kSteps steps of a tile, row (i, sub) (step i of run
// sub) at i * kSub + sub, so that lanes read neighbouring words.  Each warp copies
// and reads its own rows only; rows past the length and channels past D are not
// copied, and what lies there is not used.
template <typename T, int NA, int LC, int TS, int MODE>
struct Stage {
  using La = Lanes<LC, TS>;
  static_assert(MODE != kHalfWords || sizeof(T) == 2, "fp32 rows are whole words");
  static constexpr bool kPairs = MODE == kVectors || (MODE == kWords && sizeof(T) == 2);
  // bytes; a row that starts in the middle of a word has one word more
  static constexpr int kRow = La::kTile * (int)sizeof(T) + (MODE == kHalfWords ? 4 : 0);
  static constexpr int kArray = (La::kSteps * kRow + 15) / 16 * 16;
  static constexpr int kBytes = NA * kArray;                       // per warp
  static constexpr int V = 16 / (int)sizeof(T), PR = La::kTile / V, RI = 32 / PR;
  const T* p[NA];                    // of step t0 of the row: this lane's first piece
  const T* lo[NA]; const T* hi[NA];  // kHalfWords: the array's bounds

  __device__ __forceinline__ void word(unsigned s, const void* g) const {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(s), "l"(g) : "memory");
  }
  static __device__ __forceinline__ int row_at(int rr) {
    return (rr % TS * La::kSub + rr / TS) * kRow;
  }

  // rows t0 .. below n; channels c0 .. below D
  __device__ __forceinline__ void issue(char* buf, const long long (&ld)[NA], int t0, int n,
                                        int c0, int D) const {
    const int lane = threadIdx.x;
    const unsigned to = (unsigned)__cvta_generic_to_shared(buf);
    if constexpr (MODE == kVectors) {
      const int row = lane / PR, c = lane % PR * V;
      if (c0 + c < D) {
#pragma unroll
        for (int i = 0; i < La::kSteps / RI; ++i) {
          const int rr = i * RI + row;
          if (t0 + rr < n) {
            const unsigned s = to + row_at(rr) + c * (int)sizeof(T);
#pragma unroll
            for (int k = 0; k < NA; ++k)
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(s + k * kArray),
                           "l"(p[k] + (long long)(i * RI) * ld[k])
                           : "memory");
          }
        }
      }
    } else if constexpr (MODE == kWords) {
      constexpr int E = 4 / (int)sizeof(T), W = La::kTile / E;     // elements of a word, words of a row
#pragma unroll
      for (int i = 0; i < La::kSteps * W / 32; ++i) {
        const int rr = (i * 32 + lane) / W, w = (i * 32 + lane) % W;
        if (t0 + rr < n && c0 + w * E < D) {
#pragma unroll
          for (int k = 0; k < NA; ++k)
            word(to + k * kArray + row_at(rr) + w * 4, p[k] + rr * ld[k] + w * E);
        }
      }
    } else {
      // word w of a row holds its channels 2 w and 2 w + 1, or 2 w - 1 and 2 w; a lane
      // copies the word of its first channel, and a run's last lane the one behind it
      const int sub = lane / LC, w = lane % LC, c = c0 + 2 * w;
#pragma unroll
      for (int k = 0; k < NA; ++k) {
        const T* g = p[k] + sub * TS * ld[k] + 2 * w;
        // whether a word can pass the array's ends
        const bool inside = p[k] > lo[k] && p[k] + (La::kSteps - 1) * ld[k] + La::kTile < hi[k];
#pragma unroll
        for (int i = 0; i < TS; ++i, g += ld[k]) {
          const uintptr_t at = reinterpret_cast<uintptr_t>(g);
          const int odd = (int)(at >> 1 & 1);
          const T* a = reinterpret_cast<const T*>(at & ~(uintptr_t)3);
          const unsigned s = to + k * kArray + row_at(sub * TS + i) + w * 4;
          if (t0 + sub * TS + i >= n || c - odd >= D) continue;
          const bool next = odd && w == LC - 1 && c + 1 < D;
          if (inside) {
            word(s, a);
            if (next) word(s + 4, a + 2);
          } else {
            T* q = reinterpret_cast<T*>(buf + (s - to));
            if (a >= lo[k]) q[0] = a[0];
            if (a + 1 < hi[k]) q[1] = a[1];
            if (next) {
              q[2] = a[2];
              if (a + 3 < hi[k]) q[3] = a[3];
            }
          }
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // p[k] for the row that starts at `row` (b L + t0), of `rows`
  __device__ __forceinline__ void at(int k, const void* base, long long row, long long rows,
                                     long long ld, int c0, int D) {
    const int lane = threadIdx.x;
    p[k] = static_cast<const T*>(base) + (row + (MODE == kVectors ? lane / PR : 0)) * ld + c0 +
           (MODE == kVectors ? lane % PR * V : 0);
    if constexpr (MODE == kHalfWords) {
      lo[k] = static_cast<const T*>(base);
      hi[k] = lo[k] + (rows - 1) * ld + D;
    }
  }
  // all but the last LEFT calls of issue are complete
  template <int LEFT = 0>
  static __device__ __forceinline__ void wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
    __syncwarp();
  }
  // Whether the rows of this lane's run start in the middle of a word: bit k for its
  // first step's, bit NA + k for whether that changes from step to step
  // (kHalfWords; row: b L + the step)
  __device__ __forceinline__ unsigned odd_rows(const void* const (&base)[NA],
                                               const long long (&ld)[NA], long long row,
                                               int c0) const {
    unsigned m = 0;
    if constexpr (MODE == kHalfWords)
#pragma unroll
      for (int k = 0; k < NA; ++k) {
        m |= (unsigned)((reinterpret_cast<uintptr_t>(base[k]) >> 1) + row * ld[k] + c0 & 1) << k;
        m |= (unsigned)(ld[k] & 1) << (NA + k);
      }
    return m;
  }
  // the lane's pair of step i of array k
  static __device__ __forceinline__ float2 get(const char* buf, int k, int i, unsigned odd) {
    const char* from = buf + k * kArray + i * La::kSub * kRow;
    if constexpr (MODE == kHalfWords) {
      const unsigned* q = reinterpret_cast<const unsigned*>(
          from + threadIdx.x / LC * kRow) + threadIdx.x % LC;
      const unsigned a = q[0], b = q[1];
      const bool o = (odd >> k ^ (odd >> (NA + k) & i)) & 1;
      return make_float2(__uint_as_float(o ? a & 0xffff0000u : a << 16),
                         __uint_as_float(o ? b << 16 : a & 0xffff0000u));
    } else {
      const Pack<T, 2> v = ld_pack<T, 2>(reinterpret_cast<const T*>(from) + 2 * threadIdx.x);
      return make_float2(v.get(0), v.get(1));
    }
  }
};

// A lane's pair of channels in a (.., D) array, element by element where a pair
// may be cut or is not aligned.
template <bool PAIR, typename T>
__device__ __forceinline__ void store_pair(T* p, float2 v, int left) {
  if constexpr (PAIR) {
    if (left > 0) {
      if constexpr (sizeof(T) == 2) *reinterpret_cast<__nv_bfloat162*>(p) = __float22bfloat162_rn(v);
      else *reinterpret_cast<float2*>(p) = v;
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
// A warp's runs, the CTA's warps and, for S > 1, the cluster's CTAs hold
// consecutive steps, forwards (DIR 1) or backwards (-1): w and rank are this warp's
// and CTA's places in that order.  A warp folds the runs ahead of its own onto the
// value before the first; the last warp passes the value behind all of them on to
// the next call.  Two buffers in turn: one CTA barrier per call.
//
// The cluster's CTAs write their runs into each other's shared memory, counted by
// an mbarrier of the receiver's (two in turn, S x LC x 16 bytes each time).  A
// cluster barrier there waits for every store to memory before it (2 x 16001 x 1280
// fp32: forward 109 against 97 us, backward 230 against 187 us).  A slot is written again two calls later, by a CTA
// that by then has this CTA's run of the call between, which was sent after every
// warp here had read the slot.  The wait is bounded: after kMbarMaxPolls polls the
// thread sets `dead`, waits no more, and the kernel records M3_ERR_DEVICE.
template <int LC>
struct Joint {
  float4* warp;      // (2, warps, LC)
  float4* cta;       // (2, S, LC), for S > 1
  float2* carry;     // (2, LC)
  uint64_t* bar;     // (2), for S > 1
  int warps, S;
  // in shared memory behind the warps' stages
  __device__ __forceinline__ Joint(char* at, int warps, int S) : warps(warps), S(S) {
    warp = reinterpret_cast<float4*>(at);
    cta = warp + 2 * warps * LC;
    carry = reinterpret_cast<float2*>(cta + (S > 1 ? 2 * S * LC : 0));
    bar = reinterpret_cast<uint64_t*>(carry + 2 * LC);
  }
  // every CTA of the cluster runs, and its barriers are set up, before any is written to
  __device__ __forceinline__ void start() const;
  __device__ __forceinline__ float4& run(int flip, int k, int cl) const {
    return warp[(flip * warps + k) * LC + cl];
  }
  __device__ __forceinline__ float4& part(int flip, int k, int cl) const {
    return cta[(flip * S + k) * LC + cl];
  }
};
inline int joint_bytes(int lanes, int warps, int S) {
  return lanes * (32 * warps + (S > 1 ? 32 * S : 0) + 16) + 16;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}
template <int LC>
__device__ __forceinline__ void Joint<LC>::start() const {
  if (S == 1) return;
  if (threadIdx.x + threadIdx.y == 0) {
    mbar_init(bar, 1);
    mbar_init(bar + 1, 1);
    mbar_fence_init();
  }
  cluster_sync();
}
__device__ __forceinline__ unsigned peer_addr(const void* p, int peer) {
  unsigned to;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_addr(p)), "r"(peer));
  return to;
}
__device__ __forceinline__ float2 shfl2(float2 v, int from) {
  return make_float2(__shfl_sync(0xffffffffu, v.x, from & 31),
                     __shfl_sync(0xffffffffu, v.y, from & 31));
}
__device__ __forceinline__ Run as_run(const float4& v) {
  return Run{make_float2(v.x, v.y), make_float2(v.z, v.w)};
}

// The value in front of this run; turn: the call's number.  first: `carry` is the value
// in front of all, else the last call's.  On return carry is the value behind all, in
// the last warp's last run's lanes.
template <int LC, int DIR>
__device__ __forceinline__ float2 join(const Joint<LC>& j, int turn, const Run& mine, int w,
                                       int rank, bool first, float2& carry, bool& dead) {
  const int flip = turn & 1;
  const int warps = j.warps, S = j.S;
  constexpr int kSub = 32 / LC;
  const int lane = threadIdx.x, cl = lane % LC;
  const int sub = DIR > 0 ? lane / LC : kSub - 1 - lane / LC;     // this run's place in the warp
  Run upto = mine, ahead{f2(1.f), f2(0.f)};                       // through this run; ahead of it
  if (kSub > 1) {
#pragma unroll
    for (int s = 1; s < kSub; s *= 2) {
      Run f{shfl2(upto.P, lane - DIR * s * LC), shfl2(upto.V, lane - DIR * s * LC)};
      if (sub >= s) {
        then(f, upto);
        upto = f;
      }
    }
    const Run f{shfl2(upto.P, lane - DIR * LC), shfl2(upto.V, lane - DIR * LC)};
    if (sub > 0) ahead = f;
  }
  if (sub == kSub - 1)
    j.run(flip, w, cl) = make_float4(upto.P.x, upto.P.y, upto.V.x, upto.V.y);
  __syncthreads();
  float2 c = first ? carry : j.carry[flip * LC + cl];
  if (S == 1) {
    for (int k = 0; k < w; ++k) {
      const Run f = as_run(j.run(flip, k, cl));
      c = fma2(f.P, c, f.V);
    }
    if (w == warps - 1) {
      carry = fma2(upto.P, c, upto.V);
      if (sub == kSub - 1) j.carry[(flip ^ 1) * LC + cl] = carry;
    }
    return kSub > 1 ? fma2(ahead.P, c, ahead.V) : c;
  }
  Run before{f2(1.f), f2(0.f)};
  for (int k = 0; k < w; ++k) then(before, as_run(j.run(flip, k, cl)));
  if (w == warps - 1) {
    if (lane == 0) mbar_arrive_expect_tx(j.bar + flip, S * LC * 16);
    if (sub == kSub - 1) {
      Run all = before;
      then(all, upto);
      for (int peer = 0; peer < S; ++peer)
        asm volatile(
            "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 "
            "[%0], {%1, %2, %3, %4}, [%5];" ::"r"(peer_addr(&j.part(flip, rank, cl), peer)),
            "f"(all.P.x), "f"(all.P.y), "f"(all.V.x), "f"(all.V.y),
            "r"(peer_addr(j.bar + flip, peer))
            : "memory");
    }
    __syncwarp();
  }
  if (!dead) dead = !mbar_wait(j.bar + flip, turn >> 1 & 1);
  for (int k = 0; k < rank; ++k) {
    const Run f = as_run(j.part(flip, k, cl));
    c = fma2(f.P, c, f.V);
  }
  if (w == warps - 1) {
    carry = c;
    for (int k = rank; k < S; ++k) {
      const Run f = as_run(j.part(flip, k, cl));
      carry = fma2(f.P, carry, f.V);
    }
    if (sub == kSub - 1) j.carry[(flip ^ 1) * LC + cl] = carry;
  }
  c = fma2(before.P, c, before.V);
  return kSub > 1 ? fma2(ahead.P, c, ahead.V) : c;
}

}  // namespace m3
