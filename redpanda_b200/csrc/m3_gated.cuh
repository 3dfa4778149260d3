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
// e^f - 1's relative error, which is 1.83e-8 at most.  On the MUFU
// unit's ex2 instead, whose results are low by 2e-8 on average, a state would be
// low by that times 1 / (1 - a): 2e-5 at a = 0.999.
//
// All pairs below are two channels in one packed register pair: with scalar
// instructions instead the forward took 82 against 75 us (256 x 64 x 2048 bf16).
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "m3_api_util.h"
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

// How rows are copied and read, by what their starts and lengths allow, always
// asynchronously: 16 bytes at a time; words (fp32, and bf16 rows of whole words); bf16 rows
// that start anywhere, 16 bytes at a time from the 16 that the first element lies in, and
// 16 more, to be read behind the row's shift in there.  With plain loads a row that is
// not aligned to 16 bytes is waited for where it is asked for (2 x 16001 x 1281 fp32: 447
// against 165 us forward, 832 against 333 backward).  Rows that start anywhere (256 x 64 x
// 2047 bf16): 103 forward and 190 backward; by words, of which two hold a lane's pair, and
// with neighbours in a pair 161 and 320.  Whole words copied as those rows are: 98 and 188
// against 76 and 146 (2046).
enum Copy { kAny = 0, kWords = 1, kVectors = 2 };

// A warp's rows of NA arrays: kSteps steps of a tile, row (i, sub) (step i of run
// sub) at i * kSub + sub, so that lanes read neighbouring words.  Each warp copies
// and reads its own rows only; rows past the length and channels past D are not
// copied, and what lies there is not used.
template <typename T, int NA, int LC, int TS, int MODE>
struct Stage {
  using La = Lanes<LC, TS>;
  static_assert(MODE != kAny || sizeof(T) == 2, "fp32 rows are whole words");
  // A lane's channels are neighbours where pairs are whole and aligned in every array, else
  // LC apart, so that accesses of one element are those of consecutive lanes.
  static constexpr bool kPairs = MODE == kVectors || (MODE == kWords && sizeof(T) == 2);
  static constexpr int kNext = kPairs ? 1 : LC;                    // to the second channel
  static constexpr int kRow = La::kTile * (int)sizeof(T) + (MODE == kAny ? 16 : 0);   // bytes
  static constexpr int kArray = La::kSteps * kRow, kBytes = NA * kArray;                  // per warp
  static constexpr int V = 16 / (int)sizeof(T), PR = La::kTile / V, RI = 32 / PR;
  static_assert(La::kSteps % RI == 0 && La::kSteps <= 32, "copies take whole rows");
  const T* p[NA];                    // of step t0 of the row: this lane's first piece
  struct Shift { unsigned at[NA], step[NA]; };        // of a run's rows, in bytes

  // a lane's first channel in the tile
  static __device__ __forceinline__ int channel() {
    return threadIdx.x % LC * (kPairs ? 2 : 1);
  }
  static __device__ __forceinline__ int row_at(int rr) {
    return (rr % TS * La::kSub + rr / TS) * kRow;
  }
  static __device__ __forceinline__ void copy16(unsigned s, uintptr_t g) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(s), "l"(g) : "memory");
  }
  // the 16 bytes at g, less what lies outside the array
  static __device__ __forceinline__ void copy_part(unsigned s, uintptr_t g, uintptr_t lo,
                                                   uintptr_t hi) {
    if (g >= lo) {
      const int n = hi - g < 16 ? (int)(hi - g) : 16;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(s), "l"(g), "r"(n)
                   : "memory");
    } else {
      for (int i = 0; i < 16; i += (int)sizeof(T))
        if (g + i >= lo && g + i < hi) {
          if constexpr (sizeof(T) == 2)
            asm volatile("st.shared.u16 [%0], %1;" ::"r"(s + i),
                         "h"(*reinterpret_cast<const unsigned short*>(g + i))
                         : "memory");
          else
            asm volatile("st.shared.u32 [%0], %1;" ::"r"(s + i),
                         "r"(*reinterpret_cast<const unsigned*>(g + i))
                         : "memory");
        }
    }
  }

  // rows t0 .. below n; channels c0 .. below D; of the arrays at base, `rows` rows each
  __device__ __forceinline__ void issue(char* buf, const void* const (&base)[NA],
                                        const long long (&ld)[NA], long long rows, int t0, int n,
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
              copy16(s + k * kArray, reinterpret_cast<uintptr_t>(p[k] + (long long)(i * RI) * ld[k]));
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
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + k * kArray +
                                                                          row_at(rr) + w * 4),
                         "l"(p[k] + rr * ld[k] + w * E)
                         : "memory");
        }
      }
    } else {
      const int row = lane / PR, width = min(D - c0, La::kTile) * (int)sizeof(T);
#pragma unroll
      for (int k = 0; k < NA; ++k) {
        const uintptr_t lo = reinterpret_cast<uintptr_t>(base[k]),
                        hi = lo + ((rows - 1) * ld[k] + D) * (long long)sizeof(T);
        const uintptr_t mine = reinterpret_cast<uintptr_t>(p[k]);
        const long long bytes = ld[k] * (long long)sizeof(T);      // from row to row
        const uintptr_t first = mine - row * bytes;                // row 0
        auto needed = [&](int rr, uintptr_t from, uintptr_t g) {
          return t0 + rr < n && g < from + width;
        };
        if ((first & ~(uintptr_t)15) >= lo && first + (La::kSteps - 1) * bytes + kRow <= hi) {
          auto copy = [&](int rr, uintptr_t from, int piece) {
            const uintptr_t g = (from & ~(uintptr_t)15) + piece * 16;
            if (needed(rr, from, g)) copy16(to + k * kArray + row_at(rr) + piece * 16, g);
          };
#pragma unroll
          for (int i = 0; i < La::kSteps / RI; ++i)
            copy(i * RI + row, mine + (long long)(i * RI) * bytes, lane % PR);
          if (lane < La::kSteps) copy(lane, first + lane * bytes, PR);
        } else {                                     // pieces may pass the array's ends
#pragma unroll 1
          for (int i = lane; i < La::kSteps * (PR + 1); i += 32) {
            const int rr = i / (PR + 1), piece = i % (PR + 1);
            const uintptr_t from = first + rr * bytes,
                            g = (from & ~(uintptr_t)15) + piece * 16;
            if (needed(rr, from, g)) copy_part(to + k * kArray + row_at(rr) + piece * 16, g, lo, hi);
          }
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // p[k] for the row that starts at `row` (b L + t0)
  __device__ __forceinline__ void at(int k, const void* base, long long row, long long ld, int c0) {
    const int lane = threadIdx.x;
    p[k] = static_cast<const T*>(base) + (row + (MODE == kWords ? 0 : lane / PR)) * ld + c0 +
           (MODE == kVectors ? lane % PR * V : 0);
  }
  // all but the last LEFT calls of issue are complete
  template <int LEFT = 0>
  static __device__ __forceinline__ void wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
    __syncwarp();
  }
  // of this lane's run, whose first step is row b L + t
  static __device__ __forceinline__ Shift shifts(const void* const (&base)[NA],
                                                 const long long (&ld)[NA], long long row,
                                                 int c0) {
    Shift m = {};
    if constexpr (MODE == kAny)
#pragma unroll
      for (int k = 0; k < NA; ++k) {
        m.step[k] = (unsigned)ld[k] * (unsigned)sizeof(T);
        m.at[k] = (unsigned)reinterpret_cast<uintptr_t>(base[k]) + (unsigned)row * m.step[k] +
                  c0 * (unsigned)sizeof(T);
      }
    return m;
  }
  // the lane's pair of step i of array k
  static __device__ __forceinline__ float2 get(const char* buf, int k, int i, const Shift& m) {
    const char* from = buf + k * kArray + i * La::kSub * kRow;
    if constexpr (kPairs) {
      const Pack<T, 2> v = ld_pack<T, 2>(reinterpret_cast<const T*>(from) + 2 * threadIdx.x);
      return make_float2(v.get(0), v.get(1));
    } else {
      const unsigned shift = MODE == kAny ? m.at[k] + i * m.step[k] & 15u : 0u;
      const T* q = reinterpret_cast<const T*>(from + threadIdx.x / LC * kRow + shift) + channel();
      return make_float2(Elem<T>::get(q[0]), Elem<T>::get(q[LC]));
    }
  }
};

// A lane's two channels in a (.., D) array, NEXT apart (St: the Stage), of which `left`
// are there from the first one on.
template <typename St, typename T>
__device__ __forceinline__ void store_pair(T* p, float2 v, int left) {
  if constexpr (St::kPairs) {
    if (left > 0) {
      if constexpr (sizeof(T) == 2) *reinterpret_cast<__nv_bfloat162*>(p) = __float22bfloat162_rn(v);
      else *reinterpret_cast<float2*>(p) = v;
    }
  } else {
    if (left > 0) p[0] = Elem<T>::put(v.x);
    if (left > St::kNext) p[St::kNext] = Elem<T>::put(v.y);
  }
}
// the same of fp32 arrays that need not be aligned to pairs
template <typename St>
__device__ __forceinline__ void store_each(float* p, float2 v, int left) {
  if (left > 0) p[0] = v.x;
  if (left > St::kNext) p[St::kNext] = v.y;
}
template <typename St>
__device__ __forceinline__ float2 load_each(const float* p, int left) {
  return make_float2(left > 0 ? p[0] : 0.f, left > St::kNext ? p[St::kNext] : 0.f);
}

// -c softplus(decay) of a lane's two channels; 0, a decay of 1, where there is none, which
// has no say in the form of the decay that a warp takes (with another value there the last
// tile's warps never took the short one: 256 x 64 x 2040 bf16 forward 60 against 58 us, 2 x
// 16001 x 1272 fp32 backward 211 against 206; 1 x 16384 x 1000 bf16 55 either way).
template <typename St>
__device__ __forceinline__ float2 rates(const float* decay, float c, int left) {
  const float2 d = load_each<St>(decay, left);
  return make_float2(left > 0 ? -c * softplus_f(d.x) : 0.f,
                     left > St::kNext ? -c * softplus_f(d.y) : 0.f);
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

// CTAs of kGatedWarps warps in clusters of k that are resident at once, 0 on an error; asked
// for once per device.
template <auto* kern>
int resident_in_clusters(OncePerDevice& known, int k, int smem) {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= kMaxDevices) { cudaGetLastError(); return 0; }
  if ((n = known.value[dev].load(std::memory_order_acquire)) > 0) return n;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = k;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(k);
  cfg.blockDim = dim3(32, kGatedWarps);
  cfg.dynamicSmemBytes = smem;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (allow_smem<kern>(smem) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  known.value[dev].store(n * k, std::memory_order_release);
  return n * k;
}

}  // namespace m3
