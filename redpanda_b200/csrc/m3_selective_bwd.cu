// Selective scan, backward (the recurrence stands in m3_selective.cuh).
//
// With gy = dy silu(z) and the state's gradient dh carried from the back:
//   dh_t  = C_t gy_t + exp(de_{t+1} A) dh_{t+1}
//   dC_t  = sum_d gy h_t              dB_t = sum_d dh_t de u
//   s1    = sum_n dh_t B_t            w = dh_t exp(de A) h_{t-1}
//   du    = D gy + de s1              d de = u s1 + sum_n w A
//   dA    = sum_{b,t} w de            ddt = d de sigmoid(dt + bias) = d de (1 - e^-de)
//   dz    = dy (C.h + D u) silu'(z)   dD = sum gy u,  dbias = sum ddt
//
// The forward leaves the state before every chunk of kSelSteps steps.  A CTA
// owns a tile of channels, walks rows of the batch and chunks from the back:
// one sweep rebuilds the states at every fourth step (kept in shared memory),
// then each group of four steps is recomputed with its gates and gate-state
// products in registers and taken back.  So a state costs 1.75 exponentials
// here, about 16 packed FMA-pipe operations per two states, and no state but
// the checkpoints moves through memory.
//
// Sums over channels (dB, dC): pairs of channels in a thread, transposed
// shuffles over a warp's lane groups, warps joined through shared memory in
// order, channel tiles as partials that a second launch adds in order.  Sums
// over rows (dA, dD, dbias) stay in registers over a CTA's rows, then partials
// too.  No atomics: results do not depend on scheduling.
//
// Few rows: the steps are split over CTAs as in the forward, with the state's
// gradient at each run's end from per-run summaries joined from the back.
#include "m3_api_util.h"
#include "m3_selective.cuh"

namespace m3 {
namespace {

constexpr int kSub = 4;                      // steps per recomputed group
constexpr int kNSub = kSelSteps / kSub;
constexpr float kLn2 = 0x1.62e43p-1f;

template <int LN> struct BwdSmem {
  using G = Sel<LN>;
  static constexpr int NW = G::NT / 32;
  float B[kS * G::NP], C[kS * G::NP];
  float4 D[kS][G::DT];                       // (de, de u, gy, -)
  float4 H[kNSub][2][G::NT];                 // states at each group's start
  float R[kS][3][G::DT];                     // s1, s2 (in units of 1/log2 e), C.h
  float BC[2][kSub][NW][2 * G::NP];          // warps' sums of dB, dC
};

// Sum over a warp's 32 / LN lane groups of 8 values per lane, transposed:
// lane l ends with 8 LN / 32 totals (at least one), the first of index
// first_bc(l).
template <int NV, int LN, int M = 16>
__device__ __forceinline__ void group_sum(float* v, int lane) {
  if constexpr (M >= LN) {
    if constexpr (NV >= 2) {
      const bool up = (lane & M) != 0;
#pragma unroll
      for (int i = 0; i < NV / 2; ++i) {
        const float keep = up ? v[NV / 2 + i] : v[i];
        const float send = up ? v[i] : v[NV / 2 + i];
        v[i] = keep + __shfl_xor_sync(0xffffffffu, send, M);
      }
      group_sum<NV / 2, LN, M / 2>(v, lane);
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], M);
      group_sum<1, LN, M / 2>(v, lane);
    }
  }
}

// SUM: only the gradient that a run hands to the run before it, and the sum of
// its step sizes.
template <typename T, int LN, bool SUM>
__global__ void __launch_bounds__(Sel<LN>::NT) sel_bwd_kernel(const SelBwdParams bp) {
  using G = Sel<LN>;
  using M = TileMap<T, LN>;
  using Sm = BwdSmem<LN>;
  const SelParams& p = bp.f;
  extern __shared__ __align__(16) unsigned char raw_smem[];
  Sm& sm = *reinterpret_cast<Sm*>(raw_smem);
  const int q = threadIdx.x % LN, grp = threadIdx.x / LN;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c0 = blockIdx.x * G::DT, c = c0 + 2 * grp, n0 = 4 * q;
  const int split = SUM ? blockIdx.y % (p.splits - 1) + 1 : blockIdx.y % p.splits;
  const int bg = SUM ? blockIdx.y / (p.splits - 1) : blockIdx.y / p.splits;
  const int ch0 = split * p.cps, ch1 = min(ch0 + p.cps, p.nch);

  float2 a2[2][2], dA[2][2];
  load_a2(a2, p.A, c, n0, p.D, p.N);
#pragma unroll
  for (int k = 0; k < 2; ++k) dA[k][0] = dA[k][1] = make_float2(0.f, 0.f);
  // a thread's staged elements share their columns
  float bias[M::VW], dsk[M::VW], dD[M::VW], dbias[M::VW];
#pragma unroll
  for (int j = 0; j < M::VW; ++j) {
    const int cc = c0 + M::col(0) + j;
    bias[j] = (p.dt_bias && cc < p.D) ? p.dt_bias[cc] : 0.f;
    dsk[j] = (p.dskip && cc < p.D) ? p.dskip[cc] : 0.f;
    dD[j] = dbias[j] = 0.f;
  }

  for (size_t b = bg; b < (size_t)p.B; b += bp.bgroups) {
    const int n = sel_length(p.lengths, (int)b, p.L);
    const size_t rows = b * p.L;
    const T* u = static_cast<const T*>(p.u) + rows * p.ld_u;
    const T* dt = static_cast<const T*>(p.dt) + rows * p.ld_dt;
    const T* z = p.z ? static_cast<const T*>(p.z) + rows * p.ld_z : nullptr;
    const T* g = static_cast<const T*>(bp.g) + rows * p.D;
    const T* Bm = static_cast<const T*>(p.Bm) + rows * p.ld_b;
    const T* Cm = static_cast<const T*>(p.Cm) + rows * p.ld_c;
    T* du = static_cast<T*>(bp.du) + rows * p.D;
    T* ddt = static_cast<T*>(bp.ddt) + rows * p.D;
    T* dz = p.z ? static_cast<T*>(bp.dz) + rows * p.D : nullptr;

    float2 dh[2][2];
    if (!SUM && bp.qin != nullptr && split + 1 < p.splits)
      load_quads(dh, bp.qin, (size_t)split * p.B + b, c, q, p.D, G::NP);
    else
#pragma unroll
      for (int k = 0; k < 2; ++k) dh[k][0] = dh[k][1] = make_float2(0.f, 0.f);
    float dsum[2] = {0.f, 0.f};

    for (int ch = ch1 - 1; ch >= ch0; --ch) {
      const int t0 = ch * kS;
      if (t0 >= n) {   // past the row's length: no gradient
        if (!SUM)
#pragma unroll
          for (int i = 0; i < M::NVEC; ++i) {
            const auto zero = zero_pack<T, M::VW>();
            store_tile<T, LN>(zero, i, du, p.D, t0, p.L, c0, p.D, p.vec_d && bp.vec_g);
            store_tile<T, LN>(zero, i, ddt, p.D, t0, p.L, c0, p.D, p.vec_d && bp.vec_g);
            if (dz) store_tile<T, LN>(zero, i, dz, p.D, t0, p.L, c0, p.D, p.vec_d && bp.vec_g);
          }
        continue;
      }
      Pack<T, M::VW> ru[M::NVEC], rg[M::NVEC], rz[M::NVEC];
      {
        Pack<T, M::VW> rd[M::NVEC];
        Pack<T, 4> nb[G::QPT], nc[G::QPT];
        load_tile<T, LN>(rd, dt, p.ld_dt, t0, n, c0, p.D, p.vec_d);
        load_tile<T, LN>(rg, g, p.D, t0, n, c0, p.D, bp.vec_g);
        if (z) load_tile<T, LN>(rz, z, p.ld_z, t0, n, c0, p.D, p.vec_d);
        load_quad_rows<T, LN>(nc, Cm, p.ld_c, t0, n, p.N, p.vec_n);
        if (!SUM) {
          load_tile<T, LN>(ru, u, p.ld_u, t0, n, c0, p.D, p.vec_d);
          load_quad_rows<T, LN>(nb, Bm, p.ld_b, t0, n, p.N, p.vec_n);
        }
#pragma unroll
        for (int i = 0; i < M::NVEC; ++i) {
          const int r = M::row(i), cc = M::col(i);
          const bool live = t0 + r < n;
#pragma unroll
          for (int j = 0; j < M::VW; ++j) {
            const float de = live ? step_size(rd[i].get(j) + bias[j], p.softplus) : 0.f;
            float gy = rg[i].get(j);
            if (z) gy *= silu_f(rz[i].get(j));
            sm.D[r][cc + j] = make_float4(de, SUM ? 0.f : de * ru[i].get(j), gy, 0.f);
          }
        }
        put_quad_rows<T, LN>(nc, sm.C);
        if (!SUM) put_quad_rows<T, LN>(nb, sm.B);
      }
      __syncthreads();
      if (SUM) {
#pragma unroll 4
        for (int t = kS - 1; t >= 0; --t) {
          const float4 cc = *reinterpret_cast<const float4*>(sm.C + t * G::NP + n0);
          const float2 c2[2] = {make_float2(cc.x, cc.y), make_float2(cc.z, cc.w)};
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float4 dd = sm.D[t][2 * grp + k];
            dsum[k] += dd.x;
#pragma unroll
            for (int j = 0; j < 2; ++j)
              dh[k][j] = __fmul2_rn(ex2_pair(__fmul2_rn(f2(dd.x), a2[k][j])),
                                    __ffma2_rn(f2(dd.z), c2[j], dh[k][j]));
          }
        }
        __syncthreads();
        continue;
      }
      // states at every group's start
      float2 h[2][2];
      if (ch > 0) load_quads(h, p.ckpt, b * (p.nch - 1) + ch - 1, c, q, p.D, G::NP);
      else load_state(h, p.h0, b, c, n0, p.D, p.N);
#pragma unroll 1
      for (int sub = 0; sub < kNSub; ++sub) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
          sm.H[sub][k][threadIdx.x] = make_float4(h[k][0].x, h[k][0].y, h[k][1].x, h[k][1].y);
        if (sub == kNSub - 1) break;
#pragma unroll
        for (int s = 0; s < kSub; ++s) {
          const int t = sub * kSub + s;
          const float4 bb = *reinterpret_cast<const float4*>(sm.B + t * G::NP + n0);
          const float2 b2[2] = {make_float2(bb.x, bb.y), make_float2(bb.z, bb.w)};
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float2 dd = *reinterpret_cast<const float2*>(&sm.D[t][2 * grp + k]);
#pragma unroll
            for (int j = 0; j < 2; ++j)
              h[k][j] = __ffma2_rn(ex2_pair(__fmul2_rn(f2(dd.x), a2[k][j])), h[k][j],
                                   __fmul2_rn(f2(dd.y), b2[j]));
          }
        }
      }
#pragma unroll 1
      for (int sub = kNSub - 1; sub >= 0; --sub) {
        float2 ga[kSub][2][2], gh[kSub][2][2];   // gate, gate * state before
        float ys[2 * kSub], ss[4 * kSub];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float4 v = sm.H[sub][k][threadIdx.x];
          h[k][0] = make_float2(v.x, v.y);
          h[k][1] = make_float2(v.z, v.w);
        }
#pragma unroll
        for (int s = 0; s < kSub; ++s) {
          const int t = sub * kSub + s;
          const float4 bb = *reinterpret_cast<const float4*>(sm.B + t * G::NP + n0);
          const float4 cc = *reinterpret_cast<const float4*>(sm.C + t * G::NP + n0);
          const float2 b2[2] = {make_float2(bb.x, bb.y), make_float2(bb.z, bb.w)};
          const float2 c2[2] = {make_float2(cc.x, cc.y), make_float2(cc.z, cc.w)};
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float2 dd = *reinterpret_cast<const float2*>(&sm.D[t][2 * grp + k]);
            float2 y2;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              ga[s][k][j] = ex2_pair(__fmul2_rn(f2(dd.x), a2[k][j]));
              gh[s][k][j] = __fmul2_rn(ga[s][k][j], h[k][j]);
              h[k][j] = __ffma2_rn(f2(dd.y), b2[j], gh[s][k][j]);
              y2 = j ? __ffma2_rn(h[k][j], c2[j], y2) : __fmul2_rn(h[k][j], c2[j]);
            }
            ys[2 * s + k] = y2.x + y2.y;
          }
        }
#pragma unroll
        for (int s = kSub - 1; s >= 0; --s) {
          const int t = sub * kSub + s;
          const float4 bb = *reinterpret_cast<const float4*>(sm.B + t * G::NP + n0);
          const float4 cc = *reinterpret_cast<const float4*>(sm.C + t * G::NP + n0);
          const float2 b2[2] = {make_float2(bb.x, bb.y), make_float2(bb.z, bb.w)};
          const float2 c2[2] = {make_float2(cc.x, cc.y), make_float2(cc.z, cc.w)};
          float2 vb[2], vc[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float4 dd = sm.D[t][2 * grp + k];
            const float2 de = f2(dd.x), deu = f2(dd.y), gy = f2(dd.z);
            float2 x1, x2;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float2 ht = __ffma2_rn(deu, b2[j], gh[s][k][j]);
              dh[k][j] = __ffma2_rn(gy, c2[j], dh[k][j]);
              vc[j] = k ? __ffma2_rn(gy, ht, vc[j]) : __fmul2_rn(gy, ht);
              vb[j] = k ? __ffma2_rn(deu, dh[k][j], vb[j]) : __fmul2_rn(deu, dh[k][j]);
              x1 = j ? __ffma2_rn(dh[k][j], b2[j], x1) : __fmul2_rn(dh[k][j], b2[j]);
              const float2 w = __fmul2_rn(dh[k][j], gh[s][k][j]);
              x2 = j ? __ffma2_rn(w, a2[k][j], x2) : __fmul2_rn(w, a2[k][j]);
              dA[k][j] = __ffma2_rn(w, de, dA[k][j]);
              dh[k][j] = __fmul2_rn(dh[k][j], ga[s][k][j]);
            }
            ss[4 * s + 2 * k] = x1.x + x1.y;
            ss[4 * s + 2 * k + 1] = x2.x + x2.y;
          }
          float v[8] = {vb[0].x, vb[0].y, vb[1].x, vb[1].y, vc[0].x, vc[0].y, vc[1].x, vc[1].y};
          group_sum<8, LN>(v, lane);
          constexpr int KEEP = LN >= 32 ? 8 : LN == 16 ? 4 : LN == 8 ? 2 : 1;
          const int v0 = LN == 2 ? lane / 4 : lane / LN * KEEP;
          float* bc = sm.BC[sub & 1][s][warp];
          if (LN != 2 || (lane & 2) == 0)
#pragma unroll
            for (int i = 0; i < KEEP; ++i)
              bc[(v0 + i) / 4 * G::NP + n0 + (v0 + i) % 4] = v[i];
        }
        // channel sums over the lane group: total (step, channel, s1 | s2)
        lane_sum<4 * kSub, LN>(ss, q);
        constexpr int K1 = 4 * kSub >= LN ? 4 * kSub / LN : 1;
        constexpr int P1 = 4 * kSub >= LN ? 1 : LN / (4 * kSub);
        if (q % P1 == 0)
#pragma unroll
          for (int i = 0; i < K1; ++i) {
            const int x = q / P1 * K1 + i;
            sm.R[sub * kSub + x / 4][x & 1][2 * grp + (x >> 1 & 1)] = ss[i];
          }
        if (z) {
          lane_sum<2 * kSub, LN>(ys, q);
          constexpr int K2 = 2 * kSub >= LN ? 2 * kSub / LN : 1;
          constexpr int P2 = 2 * kSub >= LN ? 1 : LN / (2 * kSub);
          if (q % P2 == 0)
#pragma unroll
            for (int i = 0; i < K2; ++i) {
              const int x = q / P2 * K2 + i;
              sm.R[sub * kSub + x / 2][2][2 * grp + (x & 1)] = ys[i];
            }
        }
        __syncthreads();
        for (int e = threadIdx.x; e < kSub * 2 * G::NP; e += G::NT) {
          const int s = e / (2 * G::NP), x = e % (2 * G::NP), t = t0 + sub * kSub + s;
          float v = sm.BC[sub & 1][s][0][x];
#pragma unroll
          for (int w = 1; w < Sm::NW; ++w) v += sm.BC[sub & 1][s][w][x];
          if (t < n)
            bp.part_bc[((size_t)blockIdx.x * p.B * p.L + rows + t) * 2 * G::NP + x] = v;
        }
      }
      // the last group's barrier is behind every write of sm.R
#pragma unroll
      for (int i = 0; i < M::NVEC; ++i) {
        const int r = M::row(i), cc = M::col(i);
        Pack<T, M::VW> odu, oddt, odz;
#pragma unroll
        for (int j = 0; j < M::VW; ++j) {
          const float4 dd = sm.D[r][cc + j];
          const float s1 = sm.R[r][0][cc + j], s2 = sm.R[r][1][cc + j] * kLn2;
          const float uu = ru[i].get(j);
          odu.put(j, fmaf(dsk[j], dd.z, dd.x * s1));
          float d = fmaf(uu, s1, s2);
          if (p.softplus) d *= -expm1f(-dd.x);
          oddt.put(j, d);
          dD[j] = fmaf(dd.z, uu, dD[j]);
          dbias[j] += d;
          if (z) {
            const float zz = rz[i].get(j), yp = fmaf(dsk[j], uu, sm.R[r][2][cc + j]);
            odz.put(j, rg[i].get(j) * yp * dsilu_f(zz, sigmoid_f(zz)));
          }
        }
        const bool vec = p.vec_d && bp.vec_g;
        store_tile<T, LN>(odu, i, du, p.D, t0, p.L, c0, p.D, vec);
        store_tile<T, LN>(oddt, i, ddt, p.D, t0, p.L, c0, p.D, vec);
        if (dz) store_tile<T, LN>(odz, i, dz, p.D, t0, p.L, c0, p.D, vec);
      }
      __syncthreads();   // sm.D and sm.R are written again
    }
    if (SUM) {
      const size_t row = (size_t)split * p.B + b;
      store_quads(dh, bp.qsum, row, c, q, p.D, G::NP);
      if (q < 2 && c + q < p.D) p.dsum[row * p.D + c + q] = dsum[q];
    }
  }
  if (SUM) return;
  // partials over this CTA's rows: dA, then dD and dbias of each channel
  constexpr int PW = G::NP + 2;
  float* part = bp.part_a + (size_t)blockIdx.y * p.D * PW;
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (c + k < p.D) {
      float* o = part + (size_t)(c + k) * PW + n0;
      *reinterpret_cast<float2*>(o) = dA[k][0];
      *reinterpret_cast<float2*>(o + 2) = dA[k][1];
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
    if (c0 + x < p.D) part[(size_t)(c0 + x) * PW + G::NP + which] = v;
  }
}

// The state's gradient at every run's end, joined from the back.
__global__ void __launch_bounds__(128) sel_join_bwd_kernel(const SelBwdParams bp, int NP) {
  const SelParams& p = bp.f;
  const long long total = (long long)p.B * p.D * NP;
  const long long i = (long long)blockIdx.x * 128 + threadIdx.x;
  if (i >= total) return;
  const int n = (int)(i % NP);
  const long long bd = i / NP;
  const float a2 = n < p.N ? p.A[(size_t)(bd % p.D) * p.N + n] * kLog2e : 0.f;
  const long long sd = (long long)p.B * p.D;
  float v = 0.f;
#pragma unroll 4
  for (int s = p.splits - 1; s > 0; --s) {
    v = fmaf(ex2_approx(p.dsum[s * sd + bd] * a2), v, bp.qsum[s * total + i]);
    bp.qin[(s - 1) * total + i] = v;
  }
}

// dB and dC: the channel tiles' partials in order; rows past a length are zero.
template <typename T>
__global__ void __launch_bounds__(128) sel_reduce_bc_kernel(const SelBwdParams bp, int tiles,
                                                            int NP) {
  const SelParams& p = bp.f;
  const long long rows = (long long)p.B * p.L;
  const int per = 2 * NP / 4;
  const long long i = (long long)blockIdx.x * 128 + threadIdx.x;
  if (i >= rows * per) return;
  const long long row = i / per;
  const int x = (int)(i % per) * 4, which = x / NP, n0 = x % NP;
  if (n0 >= p.N) return;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (row % p.L < sel_length(p.lengths, (int)(row / p.L), p.L)) {
    const float* src = bp.part_bc + row * 2 * NP + x;
#pragma unroll 8
    for (int t = 0; t < tiles; ++t) {
      const float4 v = *reinterpret_cast<const float4*>(src + (size_t)t * rows * 2 * NP);
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
  }
  T* o = static_cast<T*>(which ? bp.dC : bp.dB) + row * p.N + n0;
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
cudaError_t bwd_typed(const SelBwdParams& p, cudaStream_t s) {
  using G = Sel<LN>;
  const unsigned tiles = (unsigned)((p.f.D + G::DT - 1) / G::DT);
  constexpr int smem = (int)sizeof(BwdSmem<LN>);
  auto* main = sel_bwd_kernel<T, LN, false>;
  cudaError_t e = cudaFuncSetAttribute(main, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  if (p.f.splits > 1) {
    auto* sum = sel_bwd_kernel<T, LN, true>;
    e = cudaFuncSetAttribute(sum, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    sum<<<dim3(tiles, (p.f.splits - 1) * p.bgroups), G::NT, smem, s>>>(p);
    const long long total = (long long)p.f.B * p.f.D * G::NP;
    sel_join_bwd_kernel<<<(unsigned)((total + 127) / 128), 128, 0, s>>>(p, G::NP);
  }
  main<<<dim3(tiles, p.workers), G::NT, smem, s>>>(p);
  const long long quads = (long long)p.f.B * p.f.L * (2 * G::NP / 4);
  sel_reduce_bc_kernel<T><<<(unsigned)((quads + 127) / 128), 128, 0, s>>>(p, tiles, G::NP);
  const long long na = (long long)p.f.D * (G::NP + 2);
  sel_reduce_a_kernel<<<(unsigned)((na + 127) / 128), 128, 0, s>>>(p, G::NP);
  return cudaGetLastError();
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

}  // namespace

cudaError_t launch_sel_bwd(const SelBwdParams& p, cudaStream_t s) {
  return p.f.dtype == M3_BF16 ? bwd_lanes<__nv_bfloat16>(p, s) : bwd_lanes<float>(p, s);
}

}  // namespace m3
