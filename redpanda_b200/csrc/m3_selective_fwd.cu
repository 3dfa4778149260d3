// Selective scan, forward (the recurrence stands in m3_selective.cuh).
//
// Bound by the exponentials, one per (step, channel, state) on the MUFU unit (16
// per SM and clock), with shared memory close behind: u, dt, z and y move only
// once per (step, channel).  A CTA owns 64 channels (128 for N <= 8) of one row
// and walks its steps kSelSteps at a time; the next steps' inputs are copied into
// the threads' own slots by cp.async meanwhile, so no register waits for a load.
// 256 rows x 64 steps x 1536 channels, N = 32, bf16: 277 us, of which the
// exponentials alone are 180 us at the unit's rate (MUFU 74 %, shared memory
// 64 % busy; 432 us at first, when bf16 pairs were unpacked where they were
// loaded and softplus was the library's).
//
// With few rows (a single prompt) one pass over the steps would leave most SMs
// idle, so the steps are split: a first launch gives every run its local end
// state and the sum of its step sizes, a second joins them in order,
//   h_in[s+1] = exp(A dsum[s]) h_in[s] + h_local[s],
// and the scan proper then starts each run from its own h_in.  One row of 4096
// steps x 1024 channels, N = 16, bf16: 29 + 6 + 37 us; as programmatic dependent
// launches, each starting up while the one before it drains, 70 us together
// instead of 78.
#include "m3_api_util.h"
#include "m3_pdl.cuh"
#include "m3_selective.cuh"

namespace m3 {
namespace {

// What a CTA holds in shared memory.  Two slots for u and z: one in use (they
// are read again for the output), one being filled.
template <typename T, typename G, bool SUM> struct FwdSmem {
  using M = TileMap<T, G>;
  using Tile = Pack<T, M::VW>[M::NVEC * G::NT];
  using Quads = Pack<T, 4>[G::QPT * G::NT];
  alignas(16) float4 D[kS][G::DT / 2];       // (de, de u) of two channels, at pair_at(pair);
                                             // then a step's C.h in the place of de
  alignas(16) float B[kS * G::NP], C[SUM ? 4 : kS * G::NP];
  alignas(16) Tile u[2], z[SUM ? 1 : 2], dt;
  alignas(16) Quads b, c;
};

// SUM: only the end state and the step-size sum of a run (no y).
template <typename T, int LN, bool SUM>
__global__ void __launch_bounds__(SelF<LN>::NT) sel_fwd_kernel(const SelParams p) {
  using G = SelF<LN>;
  using M = TileMap<T, G>;
  using Sm = FwdSmem<T, G, SUM>;
  constexpr int Q = G::S / 4;   // quads per lane and channel
  static_assert(M::VW % 2 == 0, "channels are staged in pairs");
  extern __shared__ __align__(16) unsigned char raw_smem[];
  Sm& sm = *reinterpret_cast<Sm*>(raw_smem);
  const int q = threadIdx.x % LN, grp = threadIdx.x / LN;
  // channel tiles of one row are neighbours: they read the same rows of B and C
  const int tiles = (p.D + G::DT - 1) / G::DT;
  const int c0 = blockIdx.x % tiles * G::DT, c = c0 + 2 * grp, n0 = G::S * q;
  const int split = blockIdx.y;
  const size_t b = blockIdx.x / tiles;
  const int n = sel_length(p.lengths, (int)b, p.L);
  const int ch0 = split * p.cps, ch1 = min(ch0 + p.cps, p.nch);
  const T* u = static_cast<const T*>(p.u) + b * p.L * p.ld_u;
  const T* dt = static_cast<const T*>(p.dt) + b * p.L * p.ld_dt;
  const T* z = p.z ? static_cast<const T*>(p.z) + b * p.L * p.ld_z : nullptr;
  const T* Bm = static_cast<const T*>(p.Bm) + b * p.L * p.ld_b;
  const T* Cm = static_cast<const T*>(p.Cm) + b * p.L * p.ld_c;
  T* y = static_cast<T*>(p.y) + b * p.L * (size_t)p.D;
  auto fetch = [&](int ch) {
    const int t0 = ch * kS;
    fetch_tile<T, G>(sm.u[ch & 1], u, p.ld_u, t0, n, c0, p.D, p.vec_d);
    fetch_tile<T, G>(sm.dt, dt, p.ld_dt, t0, n, c0, p.D, p.vec_d);
    fetch_quads<T, G>(sm.b, Bm, p.ld_b, t0, n, p.N, p.vec_n);
    if (!SUM) {
      if (z) fetch_tile<T, G>(sm.z[ch & 1], z, p.ld_z, t0, n, c0, p.D, p.vec_d);
      fetch_quads<T, G>(sm.c, Cm, p.ld_c, t0, n, p.N, p.vec_n);
    }
    copies_commit();
  };
  if (SUM) pdl_launch_dependents();
  if (ch0 * kS < n) fetch(ch0);

  const int at = pair_at<M>(grp);
  float2 a2[2][2 * Q], h[2][2 * Q];
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int i = 0; i < Q; ++i)
      set_pairs(a2[k] + 2 * i,
                powers_of(load_quad_any(p.A, 0, c + k, n0 + 4 * i, p.D, p.N)));
  if (!SUM) pdl_wait();   // all before reads inputs only; every CTA waits for the join
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int i = 0; i < Q; ++i)
      set_pairs(h[k] + 2 * i,
                SUM ? make_float4(0.f, 0.f, 0.f, 0.f)
                    : p.hin != nullptr && split > 0
                          ? load_quad_pad(p.hin, (size_t)split * p.B + b, c + k, n0 + 4 * i, p.D,
                                          G::NP)
                          : load_quad_any(p.h0, b, c + k, n0 + 4 * i, p.D, p.N));
  float bias[M::VW], dsk[M::VW];   // a thread's staged elements share their columns
#pragma unroll
  for (int j = 0; j < M::VW; ++j) {
    const int cc = c0 + M::col(0) + j;
    bias[j] = (p.dt_bias && cc < p.D) ? p.dt_bias[cc] : 0.f;
    dsk[j] = (!SUM && p.dskip && cc < p.D) ? p.dskip[cc] : 0.f;
  }
  float dsum[2] = {0.f, 0.f};
  for (int ch = ch0; ch < ch1; ++ch) {
    const int t0 = ch * kS;
    if (SUM && t0 >= n) break;
    if (!SUM && t0 >= n) {   // past the row's length: y is zero, the state stands
#pragma unroll
      for (int i = 0; i < M::NVEC; ++i)
        store_tile<T, G>(zero_pack<T, M::VW>(), i, y, p.D, t0, p.L, c0, p.D, p.vec_d);
      continue;
    }
    copies_wait();
#pragma unroll
    for (int i = 0; i < M::NVEC; ++i) {
      const int r = M::row(i), cc = M::col(i), x = i * G::NT + threadIdx.x;
      const bool live = t0 + r < n;
      const Pack<T, M::VW> cd = sm.dt[x], cu = sm.u[ch & 1][x];
#pragma unroll
      for (int j = 0; j < M::VW; j += 2) {
        const float d0 = live ? step_size(cd.get(j) + bias[j], p.softplus) : 0.f;
        const float d1 = live ? step_size(cd.get(j + 1) + bias[j + 1], p.softplus) : 0.f;
        sm.D[r][pair_at<M>((cc + j) / 2)] = make_float4(d0, d0 * cu.get(j), d1, d1 * cu.get(j + 1));
      }
    }
#pragma unroll
    for (int i = 0; i < G::QPT; ++i) {
      const int e = (int)threadIdx.x + i * G::NT;
      if (e < G::QUADS) {
        const Pack<T, 4> vb = sm.b[e];
        *reinterpret_cast<float4*>(sm.B + 4 * e) =
            make_float4(vb.get(0), vb.get(1), vb.get(2), vb.get(3));
        if (!SUM) {
          const Pack<T, 4> vc = sm.c[e];
          *reinterpret_cast<float4*>(sm.C + 4 * e) =
              make_float4(vc.get(0), vc.get(1), vc.get(2), vc.get(3));
        }
      }
    }
    __syncthreads();
    if (ch + 1 < ch1 && t0 + kS < n) fetch(ch + 1);
    if (!SUM && p.ckpt && ch > 0)
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < Q; ++i)
          store_quad_pad(quad_of(h[k] + 2 * i), p.ckpt, b * (p.nch - 1) + ch - 1, c + k,
                         n0 + 4 * i, p.D, G::NP);
    // steps of a group: enough for the two channels' totals to fill the lanes
    constexpr int GS = SUM ? 2 : (LN >= 4 ? LN / 2 : 1);
#pragma unroll(GS >= 4 ? 1 : 4 / GS)
    for (int g0 = 0; g0 < kS; g0 += GS) {
      float acc[2 * GS];
#pragma unroll
      for (int s = 0; s < GS; ++s) {
        const int t = g0 + s;
        const float4 dd = sm.D[t][at];
        float2 ys[2];
        if (SUM) {
          dsum[0] += dd.x;
          dsum[1] += dd.z;
        }
#pragma unroll
        for (int i = 0; i < Q; ++i) {
          float2 b2[2], c2[2];
          set_pairs(b2, *reinterpret_cast<const float4*>(sm.B + t * G::NP + n0 + 4 * i));
          if (!SUM) set_pairs(c2, *reinterpret_cast<const float4*>(sm.C + t * G::NP + n0 + 4 * i));
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float2 de = f2(k ? dd.z : dd.x), du = f2(k ? dd.w : dd.y);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int x = 2 * i + j;
              const float2 a = gate_pair(de, a2[k][x]);
              h[k][x] = __ffma2_rn(a, h[k][x], __fmul2_rn(du, b2[j]));
              if (!SUM)
                ys[k] = x ? __ffma2_rn(h[k][x], c2[j], ys[k]) : __fmul2_rn(h[k][x], c2[j]);
            }
          }
        }
        if (!SUM) {
          acc[2 * s] = ys[0].x + ys[0].y;
          acc[2 * s + 1] = ys[1].x + ys[1].y;
        }
      }
      if (!SUM) {
        // total q: step q / 2, channel q % 2; only this group reads its channels
        // of sm.D, and its lanes have met in the shuffles
        lane_sum<2 * GS, LN>(acc, q);
        __syncwarp();
        if constexpr (LN == 1) {
          sm.D[g0][at].x = acc[0];
          sm.D[g0][at].z = acc[1];
        } else {
          reinterpret_cast<float*>(&sm.D[g0 + (q >> 1)][at])[2 * (q & 1)] = acc[0];
        }
      }
    }
    __syncthreads();
    if (!SUM) {
#pragma unroll
      for (int i = 0; i < M::NVEC; ++i) {
        const int r = M::row(i), cc = M::col(i), x = i * G::NT + threadIdx.x;
        const bool live = t0 + r < n;
        const Pack<T, M::VW> cu = sm.u[ch & 1][x];
        Pack<T, M::VW> cz, o;
        if (z) cz = sm.z[ch & 1][x];
#pragma unroll
        for (int j = 0; j < M::VW; j += 2) {
          const float4 yy = sm.D[r][pair_at<M>((cc + j) / 2)];
          float v0 = fmaf(dsk[j], cu.get(j), yy.x), v1 = fmaf(dsk[j + 1], cu.get(j + 1), yy.z);
          if (z) {
            v0 *= silu_f(cz.get(j));
            v1 *= silu_f(cz.get(j + 1));
          }
          o.put(j, live ? v0 : 0.f);
          o.put(j + 1, live ? v1 : 0.f);
        }
        store_tile<T, G>(o, i, y, p.D, t0, p.L, c0, p.D, p.vec_d);
      }
      // a thread stages over what it has just read itself
    }
  }
  const size_t row = SUM ? (size_t)split * p.B + b : b;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
#pragma unroll
    for (int i = 0; i < Q; ++i) {
      const float4 v = quad_of(h[k] + 2 * i);
      if (SUM) store_quad_pad(v, p.hsum, row, c + k, n0 + 4 * i, p.D, G::NP);
      else if (p.h_last != nullptr && split == p.splits - 1)
        store_quad_any(v, p.h_last, row, c + k, n0 + 4 * i, p.D, p.N);
    }
    if (SUM && q == 0 && c + k < p.D) p.dsum[row * p.D + c + k] = dsum[k];
  }
}

// h_in of every run from the runs' summaries, in order.
__global__ void __launch_bounds__(128) sel_join_kernel(const SelParams p, int NP) {
  const long long total = (long long)p.B * p.D * NP;
  const long long i = (long long)blockIdx.x * 128 + threadIdx.x;
  pdl_launch_dependents();
  if (i >= total) {
    pdl_wait();
    return;
  }
  const int n = (int)(i % NP);
  const long long bd = i / NP;
  const int d = (int)(bd % p.D);
  float h = 0.f, a2 = 0.f;
  if (n < p.N) {
    a2 = power_of(p.A[(size_t)d * p.N + n]);
    if (p.h0 != nullptr) h = p.h0[bd * p.N + n];
  }
  pdl_wait();
  const long long sd = (long long)p.B * p.D;
  constexpr int U = 32;   // runs whose summaries are loaded ahead of the chain (8: 9.0 us
                          // against 6.4 at 1 x 4096 x 1024, N = 16)
  for (int s0 = 0; s0 + 1 < p.splits; s0 += U) {
    float d[U], x[U];
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (s0 + k + 1 < p.splits) {
        d[k] = p.dsum[(s0 + k) * sd + bd];
        x[k] = p.hsum[(s0 + k) * total + i];
      }
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (s0 + k + 1 < p.splits) {
        h = carry_over(d[k] * a2, h, x[k]);
        p.hin[(s0 + k + 1) * total + i] = h;
      }
  }
}

template <typename T, int LN, bool SUM>
cudaError_t fwd_launch(const SelParams& p, int runs, bool pdl, cudaStream_t s) {
  using G = SelF<LN>;
  constexpr int smem = (int)sizeof(FwdSmem<T, G, SUM>);
  constexpr auto* kern = sel_fwd_kernel<T, LN, SUM>;
  const cudaError_t e = allow_smem<kern>(smem);
  if (e != cudaSuccess) return e;
  const unsigned tiles = (unsigned)((p.D + G::DT - 1) / G::DT);
  return launch_maybe_pdl(pdl, kern, dim3(tiles * p.B, runs), dim3(G::NT), smem, s, p);
}

template <typename T, int LN>
cudaError_t fwd_typed(const SelParams& p, cudaStream_t s) {
  using G = SelF<LN>;
  if (p.splits > 1) {
    cudaError_t e = fwd_launch<T, LN, true>(p, p.splits - 1, false, s);
    if (e != cudaSuccess) return e;
    const long long total = (long long)p.B * p.D * G::NP;
    e = launch_maybe_pdl(true, sel_join_kernel, dim3((unsigned)((total + 127) / 128)), dim3(128),
                         0, s, p, (int)G::NP);
    if (e != cudaSuccess) return e;
  }
  return fwd_launch<T, LN, false>(p, p.splits, p.splits > 1, s);
}

template <typename T, int LN>
int resident() {
  static OncePerDevice known;
  static_assert(SelF<LN>::DT == (LN == 1 ? 128 : 64), "sel_fwd_tile");
  constexpr int smem = (int)sizeof(FwdSmem<T, SelF<LN>, false>);
  return resident_ctas<sel_fwd_kernel<T, LN, false>>(known, SelF<LN>::NT, smem);
}
template <typename T>
int resident_lanes(int N) {
  switch (sel_lanes(N) / 2) {
    case 1: return resident<T, 1>();
    case 2: return resident<T, 2>();
    case 4: return resident<T, 4>();
    case 8: return resident<T, 8>();
    default: return resident<T, 16>();
  }
}

template <typename T>
cudaError_t fwd_lanes(const SelParams& p, cudaStream_t s) {
  switch (sel_lanes(p.N) / 2) {   // eight states per lane
    case 1: return fwd_typed<T, 1>(p, s);
    case 2: return fwd_typed<T, 2>(p, s);
    case 4: return fwd_typed<T, 4>(p, s);
    case 8: return fwd_typed<T, 8>(p, s);
    default: return fwd_typed<T, 16>(p, s);
  }
}

}  // namespace

int sel_fwd_resident(int N, int dtype) {
  return dtype == M3_BF16 ? resident_lanes<__nv_bfloat16>(N) : resident_lanes<float>(N);
}

cudaError_t launch_sel_fwd(const SelParams& p, cudaStream_t s) {
  return p.dtype == M3_BF16 ? fwd_lanes<__nv_bfloat16>(p, s) : fwd_lanes<float>(p, s);
}

}  // namespace m3
