// Selective scan, forward (the recurrence stands in m3_selective.cuh).
//
// Bound by the exponentials: one per (step, channel, state) on the MUFU unit
// (16 per SM and clock) beside four packed FMA-pipe operations per two states,
// while u, dt, z and y move only once per (step, channel).  A CTA owns a tile
// of channels of one row and walks its steps; raw inputs of the next kSelSteps
// steps are loaded into registers while the present ones are computed.
//
// With few rows (a single prompt) one pass over the steps would leave most SMs
// idle, so the steps are split: a first launch gives every run its local end
// state and the sum of its step sizes, a second joins them in order,
//   h_in[s+1] = exp(A dsum[s]) h_in[s] + h_local[s],
// and the scan proper then starts each run from its own h_in.
#include "m3_api_util.h"
#include "m3_selective.cuh"

namespace m3 {
namespace {

// What a CTA holds in shared memory.  Two slots per tensor: one in use (u and z
// are read again for the output), one being filled.
template <typename T, int LN, bool SUM> struct FwdSmem {
  using G = Sel<LN>;
  using M = TileMap<T, LN>;
  using Tile = Pack<T, M::VW>[M::NVEC * G::NT];
  using Quads = Pack<T, 4>[G::QPT * G::NT];
  alignas(16) float2 D[kS][G::DT];           // (de, de u)
  alignas(16) float B[kS * G::NP], C[SUM ? 4 : kS * G::NP];
  alignas(16) float Y[SUM ? 1 : kS][SUM ? 4 : G::DT];
  alignas(16) Tile u[2], z[SUM ? 1 : 2], dt;
  alignas(16) Quads b, c;
};

// SUM: only the end state and the step-size sum of a run (no y).
template <typename T, int LN, bool SUM>
__global__ void __launch_bounds__(Sel<LN>::NT) sel_fwd_kernel(const SelParams p) {
  using G = Sel<LN>;
  using M = TileMap<T, LN>;
  using Sm = FwdSmem<T, LN, SUM>;
  constexpr int TG = LN / 2;    // steps whose 2-channel totals fill the group's lanes
  extern __shared__ __align__(16) unsigned char raw_smem[];
  Sm& sm = *reinterpret_cast<Sm*>(raw_smem);
  const int q = threadIdx.x % LN, grp = threadIdx.x / LN;
  // channel tiles of one row are neighbours: they read the same rows of B and C
  const int tiles = (p.D + G::DT - 1) / G::DT;
  const int c0 = blockIdx.x % tiles * G::DT, c = c0 + 2 * grp, n0 = 4 * q;
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
    fetch_tile<T, LN>(sm.u[ch & 1], u, p.ld_u, t0, n, c0, p.D, p.vec_d);
    fetch_tile<T, LN>(sm.dt, dt, p.ld_dt, t0, n, c0, p.D, p.vec_d);
    fetch_quads<T, LN>(sm.b, Bm, p.ld_b, t0, n, p.N, p.vec_n);
    if (!SUM) {
      if (z) fetch_tile<T, LN>(sm.z[ch & 1], z, p.ld_z, t0, n, c0, p.D, p.vec_d);
      fetch_quads<T, LN>(sm.c, Cm, p.ld_c, t0, n, p.N, p.vec_n);
    }
    copies_commit();
  };
  if (ch0 * kS < n) fetch(ch0);

  float2 a2[2][2], h[2][2];
  load_a2(a2, p.A, c, n0, p.D, p.N);
  if (SUM) {
#pragma unroll
    for (int k = 0; k < 2; ++k) h[k][0] = h[k][1] = make_float2(0.f, 0.f);
  } else if (p.hin != nullptr && split > 0) {
    load_quads(h, p.hin, (size_t)split * p.B + b, c, q, p.D, G::NP);
  } else {
    load_state(h, p.h0, b, c, n0, p.D, p.N);
  }
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
        store_tile<T, LN>(zero_pack<T, M::VW>(), i, y, p.D, t0, p.L, c0, p.D, p.vec_d);
      continue;
    }
    copies_wait();
#pragma unroll
    for (int i = 0; i < M::NVEC; ++i) {
      const int r = M::row(i), cc = M::col(i), x = i * G::NT + threadIdx.x;
      const bool live = t0 + r < n;
      const Pack<T, M::VW> cd = sm.dt[x], cu = sm.u[ch & 1][x];
#pragma unroll
      for (int j = 0; j < M::VW; ++j) {
        const float de = live ? step_size(cd.get(j) + bias[j], p.softplus) : 0.f;
        const float du = live ? de * cu.get(j) : 0.f;
        sm.D[r][cc + j] = make_float2(de, du);
      }
    }
#pragma unroll
    for (int i = 0; i < G::QPT; ++i) {
      const int e = (int)threadIdx.x + i * G::NT;
      if (e < kS * LN) {
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
      store_quads(h, p.ckpt, b * (p.nch - 1) + ch - 1, c, q, p.D, G::NP);
    // steps of a group: enough for the totals to fill the lanes
    constexpr int GS = SUM ? 4 : TG;
#pragma unroll(SUM || TG >= 4 ? 1 : 4 / TG)
    for (int g0 = 0; g0 < kS; g0 += GS) {
      float acc[2 * GS];
#pragma unroll
      for (int s = 0; s < GS; ++s) {
        const int t = g0 + s;
        const float4 dd = *reinterpret_cast<const float4*>(&sm.D[t][2 * grp]);
        const float4 bb = *reinterpret_cast<const float4*>(sm.B + t * G::NP + n0);
        const float2 b2[2] = {make_float2(bb.x, bb.y), make_float2(bb.z, bb.w)};
        float2 c2[2];
        if (!SUM) {
          const float4 cc = *reinterpret_cast<const float4*>(sm.C + t * G::NP + n0);
          c2[0] = make_float2(cc.x, cc.y);
          c2[1] = make_float2(cc.z, cc.w);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float2 de = f2(k ? dd.z : dd.x), du = f2(k ? dd.w : dd.y);
          float2 ysum;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float2 a = ex2_pair(__fmul2_rn(de, a2[k][j]));
            h[k][j] = __ffma2_rn(a, h[k][j], __fmul2_rn(du, b2[j]));
            if (!SUM) ysum = j ? __ffma2_rn(h[k][j], c2[j], ysum) : __fmul2_rn(h[k][j], c2[j]);
          }
          if (SUM) dsum[k] += k ? dd.z : dd.x;
          else acc[2 * s + k] = ysum.x + ysum.y;
        }
      }
      if (!SUM) {
        lane_sum<2 * GS, LN>(acc, q);   // total q: step q / 2, channel q % 2
        sm.Y[g0 + (q >> 1)][2 * grp + (q & 1)] = acc[0];
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
        for (int j = 0; j < M::VW; ++j) {
          float v = fmaf(dsk[j], cu.get(j), sm.Y[r][cc + j]);
          if (z) v *= silu_f(cz.get(j));
          o.put(j, live ? v : 0.f);
        }
        store_tile<T, LN>(o, i, y, p.D, t0, p.L, c0, p.D, p.vec_d);
      }
      // the next chunk's barrier stands before sm.Y is written again
    }
  }
  if (SUM) {
    const size_t row = (size_t)split * p.B + b;
    store_quads(h, p.hsum, row, c, q, p.D, G::NP);
    if (q < 2 && c + q < p.D) p.dsum[row * p.D + c + q] = q ? dsum[1] : dsum[0];
  } else if (p.h_last != nullptr && split == p.splits - 1) {
    store_state(h, p.h_last, b, c, n0, p.D, p.N);
  }
}

// h_in of every run from the runs' summaries, in order.
__global__ void __launch_bounds__(128) sel_join_kernel(const SelParams p, int NP) {
  const long long total = (long long)p.B * p.D * NP;
  const long long i = (long long)blockIdx.x * 128 + threadIdx.x;
  if (i >= total) return;
  const int n = (int)(i % NP);
  const long long bd = i / NP;
  const int d = (int)(bd % p.D);
  float h = 0.f, a2 = 0.f;
  if (n < p.N) {
    a2 = p.A[(size_t)d * p.N + n] * kLog2e;
    if (p.h0 != nullptr) h = p.h0[bd * p.N + n];
  }
  const long long sd = (long long)p.B * p.D;
#pragma unroll 4
  for (int s = 0; s + 1 < p.splits; ++s) {
    h = fmaf(ex2_approx(p.dsum[s * sd + bd] * a2), h, p.hsum[s * total + i]);
    p.hin[(s + 1) * total + i] = h;
  }
}

template <typename T, int LN, bool SUM>
cudaError_t fwd_launch(const SelParams& p, int runs, cudaStream_t s) {
  using G = Sel<LN>;
  constexpr int smem = (int)sizeof(FwdSmem<T, LN, SUM>);
  constexpr auto* kern = sel_fwd_kernel<T, LN, SUM>;
  const cudaError_t e = allow_smem<kern>(smem);
  if (e != cudaSuccess) return e;
  const unsigned tiles = (unsigned)((p.D + G::DT - 1) / G::DT);
  kern<<<dim3(tiles * p.B, runs), G::NT, smem, s>>>(p);
  return cudaGetLastError();
}

template <typename T, int LN>
cudaError_t fwd_typed(const SelParams& p, cudaStream_t s) {
  using G = Sel<LN>;
  if (p.splits > 1) {
    const cudaError_t e = fwd_launch<T, LN, true>(p, p.splits - 1, s);
    if (e != cudaSuccess) return e;
    const long long total = (long long)p.B * p.D * G::NP;
    sel_join_kernel<<<(unsigned)((total + 127) / 128), 128, 0, s>>>(p, G::NP);
  }
  return fwd_launch<T, LN, false>(p, p.splits, s);
}

template <typename T>
cudaError_t fwd_lanes(const SelParams& p, cudaStream_t s) {
  switch (sel_lanes(p.N)) {
    case 2: return fwd_typed<T, 2>(p, s);
    case 4: return fwd_typed<T, 4>(p, s);
    case 8: return fwd_typed<T, 8>(p, s);
    case 16: return fwd_typed<T, 16>(p, s);
    default: return fwd_typed<T, 32>(p, s);
  }
}

}  // namespace

// Runs of the time split: enough CTAs for four per SM, when the rows and
// channel tiles alone give fewer than two.
int sel_splits(int B, int L, int D, int N, int sms) {
  const int ln = sel_lanes(N);
  const long long ctas = (long long)B * ((D + sel_tile(ln) - 1) / sel_tile(ln));
  const int nch = (L + kSelSteps - 1) / kSelSteps;
  if (ctas >= 2LL * sms || nch < 4) return 1;
  long long s = 4LL * sms / ctas;
  if (s > nch / 2) s = nch / 2;
  if (s < 2) return 1;
  const int cps = (int)((nch + s - 1) / s);
  return (nch + cps - 1) / cps;
}

cudaError_t launch_sel_fwd(const SelParams& p, cudaStream_t s) {
  return p.dtype == M3_BF16 ? fwd_lanes<__nv_bfloat16>(p, s) : fwd_lanes<float>(p, s);
}

}  // namespace m3
