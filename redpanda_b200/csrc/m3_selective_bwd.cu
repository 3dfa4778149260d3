// Selective scan, backward (the recurrence stands in m3_selective.cuh).
//
// With gy = dy silu(z) and the state's gradient dh carried from the back:
//   dh_t  = C_t gy_t + exp(de_{t+1} A) dh_{t+1}
//   dC_t  = sum_d gy h_t              dB_t = sum_d dh_t de u
//   s1    = sum_n dh_t B_t            w = dh_t exp(de A) h_{t-1}
//   du    = D gy + de s1              d de = u s1 + sum_n w A
//   dA    = sum_{b,t} w de            ddt = d de sigmoid(dt + bias)
//   dz    = dy (C.h + D u) silu'(z)   dD = sum gy u,  dbias = sum ddt
//
// The forward leaves the state before every chunk of kSelSteps steps.  A CTA
// owns a tile of channels, walks rows of the batch and chunks from the back:
// one sweep rebuilds the states at every fourth step (kept in shared memory),
// then each group of four steps is recomputed with its gates and gate-state
// products in registers and taken back.  So a state costs 1.75 exponentials
// here, about 16 packed FMA-pipe operations per two states, and no state but
// the checkpoints moves through memory.  256 rows x 64 steps x 1536 channels,
// N = 32, bf16: 1041 us (1714 us at first), with no unit above 60 % busy (issue
// 56 %, shared memory 59 %, FMA pipe 45 %, MUFU 37 %) and eleven warps per SM,
// which the registers of four steps' gates and products leave room for.
//
// Sums over channels (dB, dC): pairs of channels in a thread, transposed
// shuffles over a warp's lane groups (Order below), warps joined through shared
// memory in order, channel tiles as partials that a second launch adds in order.
// Sums over rows (dA, dD, dbias) stay in registers over a CTA's rows, then partials
// too.  No atomics: results do not depend on scheduling.  The channel tiles'
// partials are 8 NP bytes per tile and step (NP the padded states), so a large
// batch is taken in slabs of rows that share one buffer.
//
// Few rows: the steps are split over CTAs as in the forward, with the state's
// gradient at each run's end from per-run summaries joined from the back.
#include "m3_api_util.h"
#include "m3_pdl.cuh"
#include "m3_selective.cuh"

namespace m3 {
namespace {

constexpr int kSub = 4;                      // steps per recomputed group
constexpr int kNSub = kSelSteps / kSub;
constexpr float kLn2 = 0x1.62e43p-1f;

// Sums over the warp's 32 / LN lane groups (dB, dC) without selects: the halves
// of a transposed reduction are chosen by the order in which a lane holds its
// states.  Lanes with bit 4 set hold their two pairs swapped, lanes with bit 3
// set the members of each pair (as far as there are groups to add), so that a
// lane always keeps its first and sends its second half.  B and C are staged in
// every order that occurs.
template <int LN> struct Order {
  static constexpr int GROUPS = 32 / LN;
  static constexpr int COPIES = GROUPS >= 4 ? 4 : GROUPS;   // of B and C
  static __device__ __forceinline__ int pair(int lane) { return GROUPS >= 2 ? lane >> 4 & 1 : 0; }
  static __device__ __forceinline__ int elem(int lane) { return GROUPS >= 4 ? lane >> 3 & 1 : 0; }
};

template <typename T, int LN> struct BwdSmem {
  using G = Sel<LN>;
  using M = TileMap<T, Sel<LN>>;
  using Tile = Pack<T, M::VW>[M::NVEC * G::NT];
  using Quads = Pack<T, 4>[G::QPT * G::NT];
  static constexpr int NW = G::NT / 32, CP = Order<LN>::COPIES;
  alignas(16) float B[CP][kS * G::NP], C[CP][kS * G::NP];
  alignas(16) float2 D[kS][G::DT];           // (de, de u), at chan_at(channel)
  alignas(16) float Y[kS][G::DT];            // gy
  alignas(16) float P[G::EPT][G::NT];        // a thread's own: the step sizes' slopes
  alignas(16) float4 H[kNSub][2][G::NT];     // states at each group's start
  // s1, s2 (in units of 1/log2 e), C.h; the padding spreads a warp's steps over
  // the banks
  alignas(16) float R[kS][3][G::DT + 8];
  alignas(16) float BC[2][kSub][NW][2 * G::NP];   // warps' sums of dB, dC
  alignas(16) Tile u[2], z[2], g[2], dt;
  alignas(16) Quads b, c;
};

// Where a channel of a staged row stands (pairs as pair_at places them).
template <typename M>
__device__ __forceinline__ int chan_at(int c) {
  return 2 * pair_at<M>(c / 2) + (c & 1);
}

// A quad in a lane's order, and back.
__device__ __forceinline__ float4 reorder(float4 v, int pair, int elem) {
  if (pair) v = make_float4(v.z, v.w, v.x, v.y);
  if (elem) v = make_float4(v.y, v.x, v.w, v.z);
  return v;
}
__device__ __forceinline__ float2 shfl_pair(float2 v, int m) {
  return make_float2(__shfl_xor_sync(0xffffffffu, v.x, m), __shfl_xor_sync(0xffffffffu, v.y, m));
}

// The chunk's staged values from the thread's slots (t0: first step).
template <typename T, int LN>
__device__ __forceinline__ void bwd_stage(BwdSmem<T, LN>& sm, const SelParams& p, int buf, int t0,
                                          int n, bool gate,
                                          const float (&bias)[TileMap<T, Sel<LN>>::VW]) {
  using G = Sel<LN>;
  using M = TileMap<T, Sel<LN>>;
#pragma unroll
  for (int i = 0; i < M::NVEC; ++i) {
    const int r = M::row(i), cc = M::col(i), x = i * G::NT + threadIdx.x;
    const bool live = t0 + r < n;
    const Pack<T, M::VW> cd = sm.dt[x], cg = sm.g[buf][x], cu = sm.u[buf][x];
    Pack<T, M::VW> cz;
    if (gate) cz = sm.z[buf][x];
#pragma unroll
    for (int j = 0; j < M::VW; ++j) {
      float slope = 0.f;
      const float de = live ? step_size(cd.get(j) + bias[j], p.softplus, &slope) : 0.f;
      float gy = cg.get(j);
      if (gate) gy *= silu_f(cz.get(j));
      sm.D[r][chan_at<M>(cc + j)] = make_float2(de, de * cu.get(j));
      sm.Y[r][cc + j] = gy;
      sm.P[i * M::VW + j][threadIdx.x] = slope;
    }
  }
#pragma unroll
  for (int i = 0; i < G::QPT; ++i) {
    const int e = (int)threadIdx.x + i * G::NT;
    if (e < G::QUADS) {
      const Pack<T, 4> vb = sm.b[e], vc = sm.c[e];
      const float4 b4 = make_float4(vb.get(0), vb.get(1), vb.get(2), vb.get(3));
      const float4 c4 = make_float4(vc.get(0), vc.get(1), vc.get(2), vc.get(3));
#pragma unroll
      for (int k = 0; k < Order<LN>::COPIES; ++k) {
        const int pair = Order<LN>::COPIES >= 4 ? k >> 1 : k;
        const int elem = Order<LN>::COPIES >= 4 ? k & 1 : 0;
        *reinterpret_cast<float4*>(sm.C[k] + 4 * e) = reorder(c4, pair, elem);
        *reinterpret_cast<float4*>(sm.B[k] + 4 * e) = reorder(b4, pair, elem);
      }
    }
  }
}

// A row's tensors.
template <typename T> struct RowPtrs {
  const T *u, *dt, *z, *g, *B, *C;
  __device__ __forceinline__ RowPtrs(const SelBwdParams& bp, size_t rows) {
    const SelParams& p = bp.f;
    u = static_cast<const T*>(p.u) + rows * p.ld_u;
    dt = static_cast<const T*>(p.dt) + rows * p.ld_dt;
    z = p.z ? static_cast<const T*>(p.z) + rows * p.ld_z : nullptr;
    g = static_cast<const T*>(bp.g) + rows * p.D;
    B = static_cast<const T*>(p.Bm) + rows * p.ld_b;
    C = static_cast<const T*>(p.Cm) + rows * p.ld_c;
  }
};

template <typename T, int LN>
__device__ __forceinline__ void bwd_fetch(BwdSmem<T, LN>& sm, const SelBwdParams& bp,
                                          const RowPtrs<T>& r, int buf, int t0, int n, int c0) {
  using G = Sel<LN>;
  const SelParams& p = bp.f;
  fetch_tile<T, G>(sm.dt, r.dt, p.ld_dt, t0, n, c0, p.D, p.vec_d);
  fetch_tile<T, G>(sm.g[buf], r.g, p.D, t0, n, c0, p.D, bp.vec_g);
  if (r.z) fetch_tile<T, G>(sm.z[buf], r.z, p.ld_z, t0, n, c0, p.D, p.vec_d);
  fetch_quads<T, G>(sm.c, r.C, p.ld_c, t0, n, p.N, p.vec_n);
  fetch_tile<T, G>(sm.u[buf], r.u, p.ld_u, t0, n, c0, p.D, p.vec_d);
  fetch_quads<T, G>(sm.b, r.B, p.ld_b, t0, n, p.N, p.vec_n);
  copies_commit();
}

// Registers per thread: three CTAs of 128 threads per SM pay for N in 17..32 (1081
// us against 1214 us with the two that 255 registers allow, 256 rows x 64 steps x
// 1536 channels, N = 32, bf16), not for N <= 16: 672 us against 692 us with three at
// N = 16, 470 us against 619 us at N = 8 (the same rows, bf16), and 306 us against
// 329 us (2 x 4001 x 1536, N = 16, fp32).  Above 32 states a CTA has 256 threads, one
// per SM: two are slower at N = 128 (64 rows, bf16: 2292 us against 2461 us; fp32:
// 1933 us against 2132 us) and at N = 64 in fp32 (128 rows: 1253 us against 1391 us),
// and faster at N = 64 in bf16 (1290 us against 1099 us), which the rule leaves out.
template <int LN> constexpr int bwd_min_ctas() { return LN == 8 ? 3 : 1; }

template <typename T, int LN>
__global__ void __launch_bounds__(Sel<LN>::NT, bwd_min_ctas<LN>())
sel_bwd_kernel(const SelBwdParams bp) {
  using G = Sel<LN>;
  using M = TileMap<T, Sel<LN>>;
  using Sm = BwdSmem<T, LN>;
  using O = Order<LN>;
  const SelParams& p = bp.f;
  extern __shared__ __align__(16) unsigned char raw_smem[];
  Sm& sm = *reinterpret_cast<Sm*>(raw_smem);
  const int q = threadIdx.x % LN, grp = threadIdx.x / LN;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c0 = blockIdx.x * G::DT, n0 = 4 * q;
  const int split = blockIdx.y % p.splits, bg = blockIdx.y / p.splits;
  const int ch0 = split * p.cps, ch1 = min(ch0 + p.cps, p.nch);
  // the lane's order of its states, and of its channels (the upper half of a
  // group's lanes takes the second channel first)
  const int pr = O::pair(lane), el = O::elem(lane), up = (q & (LN / 2)) != 0;
  const int cc2[2] = {2 * grp + up, 2 * grp + 1 - up};
  const int ca[2] = {chan_at<M>(cc2[0]), chan_at<M>(cc2[1])};
  const float* sB = sm.B[O::COPIES >= 4 ? 2 * pr + el : pr];
  const float* sC = sm.C[O::COPIES >= 4 ? 2 * pr + el : pr];

  float2 a2[2][2], dA[2][2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float4 v = load_quad_any(p.A, 0, c0 + cc2[k], n0, p.D, p.N);
    set_pairs(a2[k], reorder(powers_of(v), pr, el));
    dA[k][0] = dA[k][1] = make_float2(0.f, 0.f);
  }
  // a thread's staged elements share their columns
  float bias[M::VW], dsk[M::VW], dD[M::VW], dbias[M::VW];
#pragma unroll
  for (int j = 0; j < M::VW; ++j) {
    const int cc = c0 + M::col(0) + j;
    bias[j] = (p.dt_bias && cc < p.D) ? p.dt_bias[cc] : 0.f;
    dsk[j] = (p.dskip && cc < p.D) ? p.dskip[cc] : 0.f;
    dD[j] = dbias[j] = 0.f;
  }

  pdl_wait();   // every CTA: the join's results, and the end of what it waited for
  for (size_t b = (size_t)bp.b0 + bg; b < (size_t)bp.b0 + bp.nb; b += bp.bgroups) {
    const int n = sel_length(p.lengths, (int)b, p.L);
    const size_t rows = b * p.L;
    const RowPtrs<T> rp(bp, rows);
    const bool gate = rp.z != nullptr;
    T* du = static_cast<T*>(bp.du) + rows * p.D;
    T* ddt = static_cast<T*>(bp.ddt) + rows * p.D;
    T* dz = gate ? static_cast<T*>(bp.dz) + rows * p.D : nullptr;
    const bool vec = p.vec_d && bp.vec_g;

    // chunks past the row's length: no gradient
    int ch = ch1 - 1;
    for (; ch >= ch0 && ch * kS >= n; --ch)
#pragma unroll
      for (int i = 0; i < M::NVEC; ++i) {
        const auto zero = zero_pack<T, M::VW>();
        store_tile<T, G>(zero, i, du, p.D, ch * kS, p.L, c0, p.D, vec);
        store_tile<T, G>(zero, i, ddt, p.D, ch * kS, p.L, c0, p.D, vec);
        if (dz) store_tile<T, G>(zero, i, dz, p.D, ch * kS, p.L, c0, p.D, vec);
      }
    if (ch < ch0) continue;
    bwd_fetch<T, LN>(sm, bp, rp, ch & 1, ch * kS, n, c0);
    float2 dh[2][2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (bp.qin != nullptr && split + 1 < p.splits)
        v = load_quad_pad(bp.qin, (size_t)split * p.B + b, c0 + cc2[k], n0, p.D, G::NP);
      set_pairs(dh[k], reorder(v, pr, el));
    }

    for (; ch >= ch0; --ch) {
      const int t0 = ch * kS, buf = ch & 1;
      // the state before the chunk
      float2 h[2][2];
#pragma unroll
      for (int k = 0; k < 2; ++k)
        set_pairs(h[k], ch > 0 ? load_quad_pad(p.ckpt, b * (p.nch - 1) + ch - 1, c0 + cc2[k], n0,
                                               p.D, G::NP)
                               : load_quad_any(p.h0, b, c0 + cc2[k], n0, p.D, p.N));
      copies_wait();
      bwd_stage<T, LN>(sm, p, buf, t0, n, gate, bias);
      __syncthreads();
      if (ch > ch0) bwd_fetch<T, LN>(sm, bp, rp, buf ^ 1, t0 - kS, n, c0);
#pragma unroll
      for (int k = 0; k < 2; ++k) set_pairs(h[k], reorder(quad_of(h[k]), pr, el));
      // states at every group's start
#pragma unroll 1
      for (int sub = 0; sub < kNSub; ++sub) {
#pragma unroll
        for (int k = 0; k < 2; ++k) sm.H[sub][k][threadIdx.x] = quad_of(h[k]);
        if (sub == kNSub - 1) break;
#pragma unroll
        for (int s = 0; s < kSub; ++s) {
          const int t = sub * kSub + s;
          float2 b2[2];
          set_pairs(b2, *reinterpret_cast<const float4*>(sB + t * G::NP + n0));
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float2 dd = sm.D[t][ca[k]];
            const float2 de = f2(dd.x), deu = f2(dd.y);
#pragma unroll
            for (int j = 0; j < 2; ++j)
              h[k][j] = __ffma2_rn(gate_pair(de, a2[k][j]), h[k][j],
                                   __fmul2_rn(deu, b2[j]));
          }
        }
      }
#pragma unroll 1
      for (int sub = kNSub - 1; sub >= 0; --sub) {
        float2 ga[kSub][2][2], gh[kSub][2][2];   // gate, gate * state before
        float sy[kSub], s1[kSub], s2[kSub];      // of the lane's first channel
#pragma unroll
        for (int k = 0; k < 2; ++k) set_pairs(h[k], sm.H[sub][k][threadIdx.x]);
#pragma unroll
        for (int s = 0; s < kSub; ++s) {
          const int t = sub * kSub + s;
          float2 b2[2], c2[2];
          set_pairs(b2, *reinterpret_cast<const float4*>(sB + t * G::NP + n0));
          set_pairs(c2, *reinterpret_cast<const float4*>(sC + t * G::NP + n0));
          float ys[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float2 dd = sm.D[t][ca[k]];
            const float2 de = f2(dd.x), deu = f2(dd.y);
            float2 y2;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              ga[s][k][j] = gate_pair(de, a2[k][j]);
              gh[s][k][j] = __fmul2_rn(ga[s][k][j], h[k][j]);
              h[k][j] = __ffma2_rn(deu, b2[j], gh[s][k][j]);
              y2 = j ? __ffma2_rn(h[k][j], c2[j], y2) : __fmul2_rn(h[k][j], c2[j]);
            }
            ys[k] = y2.x + y2.y;
          }
          // the lane keeps its first channel, its partner the other one
          sy[s] = ys[0] + __shfl_xor_sync(0xffffffffu, ys[1], LN / 2);
        }
#pragma unroll
        for (int s = kSub - 1; s >= 0; --s) {
          const int t = sub * kSub + s;
          float2 b2[2], c2[2];
          set_pairs(b2, *reinterpret_cast<const float4*>(sB + t * G::NP + n0));
          set_pairs(c2, *reinterpret_cast<const float4*>(sC + t * G::NP + n0));
          float2 vb[2], vc[2];
          float x1[2], x2[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float2 dd = sm.D[t][ca[k]];
            const float2 de = f2(dd.x), deu = f2(dd.y);
            const float2 gy = f2(sm.Y[t][cc2[k]]);
            float2 y1, y2;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float2 ht = __ffma2_rn(deu, b2[j], gh[s][k][j]);
              dh[k][j] = __ffma2_rn(gy, c2[j], dh[k][j]);
              vc[j] = k ? __ffma2_rn(gy, ht, vc[j]) : __fmul2_rn(gy, ht);
              vb[j] = k ? __ffma2_rn(deu, dh[k][j], vb[j]) : __fmul2_rn(deu, dh[k][j]);
              y1 = j ? __ffma2_rn(dh[k][j], b2[j], y1) : __fmul2_rn(dh[k][j], b2[j]);
              const float2 w = __fmul2_rn(dh[k][j], gh[s][k][j]);
              y2 = j ? __ffma2_rn(w, a2[k][j], y2) : __fmul2_rn(w, a2[k][j]);
              dA[k][j] = __ffma2_rn(w, de, dA[k][j]);
              dh[k][j] = __fmul2_rn(dh[k][j], ga[s][k][j]);
            }
            x1[k] = y1.x + y1.y;
            x2[k] = y2.x + y2.y;
          }
          s1[s] = x1[0] + __shfl_xor_sync(0xffffffffu, x1[1], LN / 2);
          s2[s] = x2[0] + __shfl_xor_sync(0xffffffffu, x2[1], LN / 2);
          // sums over the warp's lane groups
          float* bc = sm.BC[sub & 1][s][warp];
          if constexpr (O::GROUPS == 1) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              *reinterpret_cast<float2*>(bc + n0 + 2 * j) = vb[j];
              *reinterpret_cast<float2*>(bc + G::NP + n0 + 2 * j) = vc[j];
            }
          } else {
            float2 pb = __fadd2_rn(vb[0], shfl_pair(vb[1], 16));
            float2 pc = __fadd2_rn(vc[0], shfl_pair(vc[1], 16));
            if constexpr (O::GROUPS == 2) {
              *reinterpret_cast<float2*>(bc + n0 + 2 * pr) = pb;
              *reinterpret_cast<float2*>(bc + G::NP + n0 + 2 * pr) = pc;
            } else {
              float eb = pb.x + __shfl_xor_sync(0xffffffffu, pb.y, 8);
              float ec = pc.x + __shfl_xor_sync(0xffffffffu, pc.y, 8);
              const int at = n0 + 2 * pr + el;
              if constexpr (O::GROUPS == 4) {
                bc[at] = eb;
                bc[G::NP + at] = ec;
              } else {   // dB to the lanes without bit 2, dC to the others
                const bool hi = (lane & 4) != 0;
                float v = (hi ? ec : eb) + __shfl_xor_sync(0xffffffffu, hi ? eb : ec, 4);
                if constexpr (O::GROUPS == 16) v += __shfl_xor_sync(0xffffffffu, v, 2);
                if (O::GROUPS < 16 || (lane & 2) == 0) bc[(hi ? G::NP : 0) + at] = v;
              }
            }
          }
        }
        // channel sums over the group's remaining lanes: halves of the steps
        constexpr int M1 = LN / 4, M2 = LN / 8;
        if constexpr (M1 >= 1) {
          const bool hi = (q & M1) != 0;
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            s1[s] = (hi ? s1[s + 2] : s1[s]) + __shfl_xor_sync(0xffffffffu, hi ? s1[s] : s1[s + 2], M1);
            s2[s] = (hi ? s2[s + 2] : s2[s]) + __shfl_xor_sync(0xffffffffu, hi ? s2[s] : s2[s + 2], M1);
            sy[s] = (hi ? sy[s + 2] : sy[s]) + __shfl_xor_sync(0xffffffffu, hi ? sy[s] : sy[s + 2], M1);
          }
        }
        if constexpr (M2 >= 1) {
          const bool hi = (q & M2) != 0;
          s1[0] = (hi ? s1[1] : s1[0]) + __shfl_xor_sync(0xffffffffu, hi ? s1[0] : s1[1], M2);
          s2[0] = (hi ? s2[1] : s2[0]) + __shfl_xor_sync(0xffffffffu, hi ? s2[0] : s2[1], M2);
          sy[0] = (hi ? sy[1] : sy[0]) + __shfl_xor_sync(0xffffffffu, hi ? sy[0] : sy[1], M2);
#pragma unroll
          for (int m = M2 / 2; m >= 1; m >>= 1) {
            s1[0] += __shfl_xor_sync(0xffffffffu, s1[0], m);
            s2[0] += __shfl_xor_sync(0xffffffffu, s2[0], m);
            sy[0] += __shfl_xor_sync(0xffffffffu, sy[0], m);
          }
        }
        {
          constexpr int KEEP = M2 >= 1 ? 1 : M1 >= 1 ? 2 : 4;   // steps per lane
          const int s0 = M2 >= 1 ? (q & M1 ? 2 : 0) + (q & M2 ? 1 : 0)
                                 : M1 >= 1 ? (q & M1 ? 2 : 0) : 0;
          if (M2 <= 1 || (q & (M2 - 1)) == 0)
#pragma unroll
            for (int i = 0; i < KEEP; ++i) {
              float (*o)[G::DT + 8] = sm.R[sub * kSub + s0 + i];
              o[0][cc2[0]] = s1[i];
              o[1][cc2[0]] = s2[i];
              o[2][cc2[0]] = sy[i];
            }
        }
        __syncthreads();
        for (int e = threadIdx.x; e < kSub * 2 * G::NP; e += G::NT) {
          const int s = e / (2 * G::NP), x = e % (2 * G::NP), t = t0 + sub * kSub + s;
          float v = sm.BC[sub & 1][s][0][x];
#pragma unroll
          for (int w = 1; w < Sm::NW; ++w) v += sm.BC[sub & 1][s][w][x];
          if (t < n)
            bp.part_bc[(((size_t)blockIdx.x * bp.nb + (b - bp.b0)) * p.L + t) * 2 * G::NP + x] = v;
        }
      }
      // the last group's barrier is behind every write of sm.R
#pragma unroll
      for (int i = 0; i < M::NVEC; ++i) {
        const int r = M::row(i), cc = M::col(i), x = i * G::NT + threadIdx.x;
        const Pack<T, M::VW> cu = sm.u[buf][x], cg = sm.g[buf][x];
        Pack<T, M::VW> cz, odu, oddt, odz;
        if (gate) cz = sm.z[buf][x];
#pragma unroll
        for (int j = 0; j < M::VW; ++j) {
          const float gy = sm.Y[r][cc + j];
          const float v1 = sm.R[r][0][cc + j], v2 = sm.R[r][1][cc + j] * kLn2;
          const float uu = cu.get(j);
          odu.put(j, fmaf(dsk[j], gy, sm.D[r][chan_at<M>(cc + j)].x * v1));
          const float d = fmaf(uu, v1, v2) * sm.P[i * M::VW + j][threadIdx.x];
          oddt.put(j, d);
          dD[j] = fmaf(gy, uu, dD[j]);
          dbias[j] += d;
          if (gate) {
            const float zz = cz.get(j), yp = fmaf(dsk[j], uu, sm.R[r][2][cc + j]);
            odz.put(j, cg.get(j) * yp * dsilu_f(zz, sigmoid_f(zz)));
          }
        }
        store_tile<T, G>(odu, i, du, p.D, t0, p.L, c0, p.D, vec);
        store_tile<T, G>(oddt, i, ddt, p.D, t0, p.L, c0, p.D, vec);
        if (dz) store_tile<T, G>(odz, i, dz, p.D, t0, p.L, c0, p.D, vec);
      }
      __syncthreads();   // sm.D and sm.R are written again
    }
  }
  // partials over this CTA's rows: dA, then dD and dbias of each channel; a later
  // slab's rows are added to those of the slabs before
  constexpr int PW = G::NP + 2;
  pdl_launch_dependents();   // not before: waiting CTAs would take room
  float* part = bp.part_a + (size_t)blockIdx.y * p.D * PW;
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (c0 + cc2[k] < p.D) {
      float* o = part + (size_t)(c0 + cc2[k]) * PW + n0;
      // the inverse order: members first, then pairs
      float4 v = quad_of(dA[k]);
      if (el) v = make_float4(v.y, v.x, v.w, v.z);
      if (pr) v = make_float4(v.z, v.w, v.x, v.y);
      if (bp.b0) {
        const float2 a = *reinterpret_cast<const float2*>(o);
        const float2 c = *reinterpret_cast<const float2*>(o + 2);
        v = make_float4(a.x + v.x, a.y + v.y, c.x + v.z, c.y + v.w);
      }
      *reinterpret_cast<float2*>(o) = make_float2(v.x, v.y);
      *reinterpret_cast<float2*>(o + 2) = make_float2(v.z, v.w);
    }
  // threads with the same columns add in order
  constexpr int RPT = G::NT / M::PER_ROW;
  float* red = reinterpret_cast<float*>(raw_smem);   // [RPT][2][DT]
  const int r = M::row(0), cc = M::col(0);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < M::VW; ++j) {
    red[(r * 2) * G::DT + cc + j] = dD[j];
    red[(r * 2 + 1) * G::DT + cc + j] = dbias[j];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 2 * G::DT; e += G::NT) {
    const int which = e / G::DT, x = e % G::DT;
    float v = 0.f;
    for (int i = 0; i < RPT; ++i) v += red[(i * 2 + which) * G::DT + x];
    if (c0 + x < p.D) {
      float* o = part + (size_t)(c0 + x) * PW + G::NP + which;
      *o = bp.b0 ? *o + v : v;
    }
  }
}

// What a run hands to the run before it (the gradient of the state it starts
// from, as if nothing came after it), and the sum of its step sizes.
template <typename T, typename G> struct SumSmem {
  using M = TileMap<T, G>;
  using Tile = Pack<T, M::VW>[M::NVEC * G::NT];
  alignas(16) float4 D[kS][G::DT / 2];       // (de, gy) of two channels, at pair_at(pair)
  alignas(16) float C[kS * G::NP];
  alignas(16) Tile z, g, dt;
  alignas(16) Pack<T, 4> c[G::QPT * G::NT];
};
template <typename T, int LN>
__global__ void __launch_bounds__(SelF<LN>::NT) sel_bwd_sum_kernel(const SelBwdParams bp) {
  using G = SelF<LN>;
  using M = TileMap<T, G>;
  using Sm = SumSmem<T, G>;
  constexpr int Q = G::S / 4;
  const SelParams& p = bp.f;
  extern __shared__ __align__(16) unsigned char raw_smem[];
  Sm& sm = *reinterpret_cast<Sm*>(raw_smem);
  const int q = threadIdx.x % LN, grp = threadIdx.x / LN;
  const int tiles = (p.D + G::DT - 1) / G::DT;
  const int c0 = blockIdx.x % tiles * G::DT, c = c0 + 2 * grp, n0 = G::S * q;
  const size_t b = blockIdx.x / tiles;
  const int split = blockIdx.y + 1;
  const int ch0 = split * p.cps, ch1 = min(ch0 + p.cps, p.nch);
  pdl_launch_dependents();
  const int n = sel_length(p.lengths, (int)b, p.L);
  const RowPtrs<T> rp(bp, b * p.L);
  const bool gate = rp.z != nullptr;
  auto fetch = [&](int t0) {
    fetch_tile<T, G>(sm.dt, rp.dt, p.ld_dt, t0, n, c0, p.D, p.vec_d);
    fetch_tile<T, G>(sm.g, rp.g, p.D, t0, n, c0, p.D, bp.vec_g);
    if (gate) fetch_tile<T, G>(sm.z, rp.z, p.ld_z, t0, n, c0, p.D, p.vec_d);
    fetch_quads<T, G>(sm.c, rp.C, p.ld_c, t0, n, p.N, p.vec_n);
    copies_commit();
  };
  int ch = min(ch1, (n + kS - 1) / kS) - 1;
  if (ch >= ch0) fetch(ch * kS);
  const int at = pair_at<M>(grp);
  float2 a2[2][2 * Q], dh[2][2 * Q];
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int i = 0; i < Q; ++i) {
      set_pairs(a2[k] + 2 * i,
                powers_of(load_quad_any(p.A, 0, c + k, n0 + 4 * i, p.D, p.N)));
      dh[k][2 * i] = dh[k][2 * i + 1] = make_float2(0.f, 0.f);
    }
  float bias[M::VW], dsum[2] = {0.f, 0.f};
#pragma unroll
  for (int j = 0; j < M::VW; ++j) {
    const int cc = c0 + M::col(0) + j;
    bias[j] = (p.dt_bias && cc < p.D) ? p.dt_bias[cc] : 0.f;
  }
  for (; ch >= ch0; --ch) {
    const int t0 = ch * kS;
    copies_wait();
#pragma unroll
    for (int i = 0; i < M::NVEC; ++i) {
      const int r = M::row(i), cc = M::col(i), x = i * G::NT + threadIdx.x;
      const bool live = t0 + r < n;
      const Pack<T, M::VW> cd = sm.dt[x], cg = sm.g[x];
      Pack<T, M::VW> cz;
      if (gate) cz = sm.z[x];
#pragma unroll
      for (int j = 0; j < M::VW; j += 2) {
        const float d0 = live ? step_size(cd.get(j) + bias[j], p.softplus) : 0.f;
        const float d1 = live ? step_size(cd.get(j + 1) + bias[j + 1], p.softplus) : 0.f;
        float g0 = cg.get(j), g1 = cg.get(j + 1);
        if (gate) {
          g0 *= silu_f(cz.get(j));
          g1 *= silu_f(cz.get(j + 1));
        }
        sm.D[r][pair_at<M>((cc + j) / 2)] = make_float4(d0, g0, d1, g1);
      }
    }
#pragma unroll
    for (int i = 0; i < G::QPT; ++i) {
      const int e = (int)threadIdx.x + i * G::NT;
      if (e < G::QUADS) {
        const Pack<T, 4> v = sm.c[e];
        *reinterpret_cast<float4*>(sm.C + 4 * e) =
            make_float4(v.get(0), v.get(1), v.get(2), v.get(3));
      }
    }
    __syncthreads();
    if (ch > ch0) fetch(t0 - kS);
#pragma unroll 2
    for (int t = kS - 1; t >= 0; --t) {
      const float4 dd = sm.D[t][at];
      dsum[0] += dd.x;
      dsum[1] += dd.z;
#pragma unroll
      for (int i = 0; i < Q; ++i) {
        float2 c2[2];
        set_pairs(c2, *reinterpret_cast<const float4*>(sm.C + t * G::NP + n0 + 4 * i));
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float2 de = f2(k ? dd.z : dd.x), gy = f2(k ? dd.w : dd.y);
#pragma unroll
          for (int j = 0; j < 2; ++j)
            dh[k][2 * i + j] =
                __fmul2_rn(gate_pair(de, a2[k][2 * i + j]),
                           __ffma2_rn(gy, c2[j], dh[k][2 * i + j]));
        }
      }
    }
    __syncthreads();
  }
  const size_t row = (size_t)split * p.B + b;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
#pragma unroll
    for (int i = 0; i < Q; ++i)
      store_quad_pad(quad_of(dh[k] + 2 * i), bp.qsum, row, c + k, n0 + 4 * i, p.D, G::NP);
    if (q == 0 && c + k < p.D) p.dsum[row * p.D + c + k] = dsum[k];
  }
}

// The state's gradient at every run's end, joined from the back.
__global__ void __launch_bounds__(128) sel_join_bwd_kernel(const SelBwdParams bp, int NP) {
  const SelParams& p = bp.f;
  const long long total = (long long)p.B * p.D * NP;
  const long long i = (long long)blockIdx.x * 128 + threadIdx.x;
  pdl_launch_dependents();
  if (i >= total) {
    pdl_wait();
    return;
  }
  const int n = (int)(i % NP);
  const long long bd = i / NP;
  const float a2 = n < p.N ? power_of(p.A[(size_t)(bd % p.D) * p.N + n]) : 0.f;
  pdl_wait();
  const long long sd = (long long)p.B * p.D;
  float v = 0.f;
  // runs whose summaries are loaded ahead of the chain (32, as forward: 3 to 7 us of
  // 180 to 480 us saved in bf16, between 6 us saved and 11 us lost in fp32)
  constexpr int U = 8;
  for (int s0 = p.splits - 1; s0 > 0; s0 -= U) {
    float d[U], x[U];
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (s0 - k > 0) {
        d[k] = p.dsum[(s0 - k) * sd + bd];
        x[k] = bp.qsum[(s0 - k) * total + i];
      }
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (s0 - k > 0) {
        v = carry_over(d[k] * a2, v, x[k]);
        bp.qin[(s0 - k - 1) * total + i] = v;
      }
  }
}

// dB and dC: the channel tiles' partials in order; rows past a length are zero.
template <typename T>
__global__ void __launch_bounds__(128) sel_reduce_bc_kernel(const SelBwdParams bp, int tiles,
                                                            int NP) {
  const SelParams& p = bp.f;
  const long long rows = (long long)bp.nb * p.L, row0 = (long long)bp.b0 * p.L;
  const int per = 2 * NP / 4;
  const long long i = (long long)blockIdx.x * 128 + threadIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  if (i >= rows * per) return;
  const long long row = i / per;
  const int x = (int)(i % per) * 4, which = x / NP, n0 = x % NP;
  if (n0 >= p.N) return;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (row % p.L < sel_length(p.lengths, bp.b0 + (int)(row / p.L), p.L)) {
    const float* src = bp.part_bc + row * 2 * NP + x;
#pragma unroll 8
    for (int t = 0; t < tiles; ++t) {
      const float4 v = *reinterpret_cast<const float4*>(src + (size_t)t * rows * 2 * NP);
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
  }
  T* o = static_cast<T*>(which ? bp.dC : bp.dB) + (row0 + row) * p.N + n0;
  const float v[4] = {s.x, s.y, s.z, s.w};
  if (p.N % 4 == 0) {
    Pack<T, 4> r;
#pragma unroll
    for (int j = 0; j < 4; ++j) r.put(j, v[j]);
    st_pack<T, 4>(o, r);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n0 + j < p.N) o[j] = Elem<T>::put(v[j]);
  }
}

// dA, dD and dbias: the workers' partials in order.
__global__ void __launch_bounds__(128) sel_reduce_a_kernel(const SelBwdParams bp, int NP) {
  const SelParams& p = bp.f;
  const int pw = NP + 2;
  const long long i = (long long)blockIdx.x * 128 + threadIdx.x;
  pdl_wait();
  if (i >= (long long)p.D * pw) return;
  const int n = (int)(i % pw);
  const long long d = i / pw;
  if (n >= p.N && n < NP) return;
  float s = 0.f;
#pragma unroll 8
  for (int w = 0; w < bp.workers; ++w) s += bp.part_a[(size_t)w * p.D * pw + i];
  if (n < NP) bp.dA[d * p.N + n] = s;
  else if (n == NP) { if (bp.dD) bp.dD[d] = s; }
  else if (bp.dbias) bp.dbias[d] = s;
}

template <typename T, int LN>
cudaError_t bwd_typed(const SelBwdParams& p0, cudaStream_t s) {
  SelBwdParams p = p0;
  using G = Sel<LN>;
  const unsigned tiles = (unsigned)((p.f.D + G::DT - 1) / G::DT);
  constexpr int smem = (int)sizeof(BwdSmem<T, LN>);
  constexpr auto* main = sel_bwd_kernel<T, LN>;
  cudaError_t e = allow_smem<main>(smem);
  if (e != cudaSuccess) return e;
  if (p.f.splits > 1) {
    using W = SelF<LN / 2>;
    constexpr int wide = (int)sizeof(SumSmem<T, W>);
    constexpr auto* sum = sel_bwd_sum_kernel<T, LN / 2>;
    e = allow_smem<sum>(wide);
    if (e != cudaSuccess) return e;
    const unsigned wtiles = (unsigned)((p.f.D + W::DT - 1) / W::DT);
    sum<<<dim3(wtiles * p.f.B, p.f.splits - 1), W::NT, wide, s>>>(p);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    const long long total = (long long)p.f.B * p.f.D * G::NP;
    e = launch_maybe_pdl(true, sel_join_bwd_kernel, dim3((unsigned)((total + 127) / 128)),
                         dim3(128), 0, s, p, (int)G::NP);
    if (e != cudaSuccess) return e;
  }
  // slab by slab of the batch: the pass, and the sum of its partials of dB and dC
  for (p.b0 = 0; p.b0 < p.f.B; p.b0 += p0.nb) {
    p.nb = p.f.B - p.b0 < p0.nb ? p.f.B - p.b0 : p0.nb;
    e = launch_maybe_pdl(p.f.splits > 1 && p.b0 == 0, main, dim3(tiles, p.workers), dim3(G::NT),
                         smem, s, p);
    if (e != cudaSuccess) return e;
    const long long quads = (long long)p.nb * p.f.L * (2 * G::NP / 4);
    e = launch_maybe_pdl(true, sel_reduce_bc_kernel<T>, dim3((unsigned)((quads + 127) / 128)),
                         dim3(128), 0, s, p, (int)tiles, (int)G::NP);
    if (e != cudaSuccess) return e;
  }
  const long long na = (long long)p.f.D * (G::NP + 2);
  return launch_maybe_pdl(true, sel_reduce_a_kernel, dim3((unsigned)((na + 127) / 128)), dim3(128),
                          0, s, p, (int)G::NP);
}

template <typename T>
cudaError_t bwd_lanes(const SelBwdParams& p, cudaStream_t s) {
  switch (sel_lanes(p.f.N)) {
    case 2: return bwd_typed<T, 2>(p, s);
    case 4: return bwd_typed<T, 4>(p, s);
    case 8: return bwd_typed<T, 8>(p, s);
    case 16: return bwd_typed<T, 16>(p, s);
    default: return bwd_typed<T, 32>(p, s);
  }
}

template <typename T, int LN>
int resident() {
  static OncePerDevice known;
  return resident_ctas<sel_bwd_kernel<T, LN>>(known, Sel<LN>::NT, (int)sizeof(BwdSmem<T, LN>));
}

template <typename T>
int resident_lanes(int N) {
  switch (sel_lanes(N)) {
    case 2: return resident<T, 2>();
    case 4: return resident<T, 4>();
    case 8: return resident<T, 8>();
    case 16: return resident<T, 16>();
    default: return resident<T, 32>();
  }
}

}  // namespace

int sel_bwd_resident(int N, int dtype) {
  return dtype == M3_BF16 ? resident_lanes<__nv_bfloat16>(N) : resident_lanes<float>(N);
}

cudaError_t launch_sel_bwd(const SelBwdParams& p, cudaStream_t s) {
  return p.f.dtype == M3_BF16 ? bwd_lanes<__nv_bfloat16>(p, s) : bwd_lanes<float>(p, s);
}

}  // namespace m3
