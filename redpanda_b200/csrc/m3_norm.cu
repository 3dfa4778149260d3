// Layer norm and RMS norm over rows of d elements, forward and backward.
//
//   mu = mean(x) (0 for RMS), v = mean((x - mu)^2), r = 1 / sqrt(v + eps)
//   xh = (x - mu) r,  y = xh w + b
//   with q = g w:  dx = r (q - mean(q) - xh mean(q xh))   (RMS: no mean(q))
//                  dw = sum over rows of g xh,  db = sum over rows of g
//
// Bound by memory: forward reads x and writes y, backward reads x and g and
// writes dx.  So every row is read once and stays on the SM between the
// statistics and the output, 8 elements per thread in registers: few of them, so
// many rows in flight.  Rows past 8192 take 32 elements per thread, more than the
// registers of 512 or 1024 threads hold beside the next row: part of them lies in
// local memory (4096 x 16384 fp32, RMS: 101 us forward, 272 us backward, 1.2 and 2.2
// times its bytes; 4096 x 8192: 47 and 87 us).  Up to 256 elements (in the forward,
// which holds less, up to 1024 at up to 32 per lane: no barriers, 74 us against 92
// us for 131072 x 768 bf16) a warp holds a row and a CTA four of them; longer rows
// have a CTA of their own.  The variance is taken from the centred values (no
// cancellation of mean(x^2) - mu^2).  The grid is persistent: weights stay with a
// thread over a CTA's rows,
// the next row's loads are issued before the present row is reduced, and the
// backward keeps the weight gradients of its columns in registers over all its
// rows.  Each CTA writes one partial row of dw (and db); a second launch adds
// the partials in a fixed order, so results do not depend on scheduling.
// 131072 rows of 768, RMS, bf16: 70 us forward (5.8 TB/s), 132 us backward
// (4.6 TB/s; 187 us with a warp per row, whose 24 columns a lane left room for 8
// warps per SM).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "m3_api_util.h"
#include "m3_ops.h"
#include "m3_pdl.cuh"
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

// MAXT: largest CTA, MINB: CTAs of that size per SM the registers are for.
template <typename TX, typename TY, int VEC, int NV, bool WARP, int MAXT, int MINB, bool RMS>
__global__ void __launch_bounds__(MAXT, MINB) norm_fwd_kernel(const NormParams p) {
  constexpr int E = VEC * NV;
  __shared__ float red[2][64];
  const int tpr = WARP ? 32 : blockDim.x, rpc = WARP ? MAXT / 32 : 1;
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x, d = p.d;
  int flip = 0;
  const TX* x = static_cast<const TX*>(p.x);
  TY* y = static_cast<TY*>(p.y);
  float w[E], b[RMS ? 1 : E];
  const long long step = (long long)gridDim.x * rpc;
  long long r = (long long)blockIdx.x * rpc + (WARP ? threadIdx.x >> 5 : 0);
  Row<TX, VEC, NV> cur;
  if (r < p.rows) cur.load(x + (size_t)r * p.ld_x, d, t, tpr);
  load_f32<VEC, NV>(w, p.w, d, t, tpr);
  if constexpr (!RMS) load_f32<VEC, NV>(b, p.b, d, t, tpr);
  const float inv_d = 1.f / (float)d;
  for (; r < p.rows; r += step) {
    Row<TX, VEC, NV> next;
    if (r + step < p.rows) next.load(x + (size_t)(r + step) * p.ld_x, d, t, tpr);
    float v[E];
#pragma unroll
    for (int k = 0; k < E; ++k) v[k] = cur.get(k);
    float mu = 0.f;
    if constexpr (!RMS) {
      float s[1] = {0.f};
#pragma unroll
      for (int k = 0; k < E; ++k) s[0] += v[k];
      row_sum<WARP>(s, red, flip);
      mu = s[0] * inv_d;
#pragma unroll
      for (int i = 0; i < NV; ++i)   // columns past d stay zero
        if ((i * tpr + t) * VEC < d)
#pragma unroll
          for (int j = 0; j < VEC; ++j) v[i * VEC + j] -= mu;
    }
    float q[1] = {0.f};
#pragma unroll
    for (int k = 0; k < E; ++k) q[0] = fmaf(v[k], v[k], q[0]);
    row_sum<WARP>(q, red, flip);
    const float rs = rsqrtf(q[0] * inv_d + p.eps);
    if (t == 0 && p.rstd != nullptr) {
      p.rstd[r] = rs;
      if (p.mean != nullptr) p.mean[r] = mu;
    }
    TY* yr = y + (size_t)r * d;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * tpr + t) * VEC;
      if (c < d) {
        Pack<TY, VEC> o;
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          o.put(j, RMS ? v[i * VEC + j] * rs * w[i * VEC + j]
                       : fmaf(v[i * VEC + j] * rs, w[i * VEC + j], b[RMS ? 0 : i * VEC + j]));
        st_pack<TY, VEC>(yr + c, o);
      }
    }
    cur = next;
  }
}

template <typename TX, typename TY, int VEC, int NV, bool WARP, int MAXT, int MINB, bool RMS>
__global__ void __launch_bounds__(MAXT, MINB) norm_bwd_kernel(const NormBwdParams p) {
  constexpr int E = VEC * NV;
  __shared__ float red[2][64];
  __shared__ float comb[WARP ? (RMS ? 1 : 2) * E * 32 : 1];   // the CTA's warps' partials
  const int tpr = WARP ? 32 : blockDim.x, rpc = WARP ? MAXT / 32 : 1;
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x, d = p.d;
  int flip = 0;
  const TX* x = static_cast<const TX*>(p.x);
  const TY* g = static_cast<const TY*>(p.g);
  TX* dx = static_cast<TX*>(p.dx);
  float w[E], dw[E], db[RMS ? 1 : E];
  const long long step = (long long)gridDim.x * rpc;
  long long r = (long long)blockIdx.x * rpc + (WARP ? threadIdx.x >> 5 : 0);
  Row<TX, VEC, NV> cx;
  Row<TY, VEC, NV> cg;
  if (r < p.rows) {
    cx.load(x + (size_t)r * p.ld_x, d, t, tpr);
    cg.load(g + (size_t)r * d, d, t, tpr);
  }
  load_f32<VEC, NV>(w, p.w, d, t, tpr);
#pragma unroll
  for (int k = 0; k < E; ++k) {
    dw[k] = 0.f;
    if constexpr (!RMS) db[k] = 0.f;
  }
  const float inv_d = 1.f / (float)d;
  for (; r < p.rows; r += step) {
    Row<TX, VEC, NV> nx;
    Row<TY, VEC, NV> ng;
    if (r + step < p.rows) {
      nx.load(x + (size_t)(r + step) * p.ld_x, d, t, tpr);
      ng.load(g + (size_t)(r + step) * d, d, t, tpr);
    }
    const float rs = p.rstd[r], mu = RMS ? 0.f : p.mean[r];
    float s[RMS ? 1 : 2];
    s[0] = 0.f;
    if constexpr (!RMS) s[1] = 0.f;
#pragma unroll
    for (int k = 0; k < E; ++k) {
      // a column past d has g = 0 and w = 0, so nothing of it is counted
      const float xh = (RMS ? cx.get(k) : cx.get(k) - mu) * rs, gk = cg.get(k), q = gk * w[k];
      s[0] = fmaf(q, xh, s[0]);
      dw[k] = fmaf(gk, xh, dw[k]);
      if constexpr (!RMS) {
        s[1] += q;
        db[k] += gk;
      }
    }
    row_sum<WARP>(s, red, flip);
    const float mx = s[0] * inv_d, mq = RMS ? 0.f : s[RMS ? 0 : 1] * inv_d;
    TX* o = dx + (size_t)r * d;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * tpr + t) * VEC;
      if (c < d) {
        Pack<TX, VEC> v;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const int k = i * VEC + j;
          const float xh = (RMS ? cx.get(k) : cx.get(k) - mu) * rs;
          v.put(j, rs * (fmaf(cg.get(k), w[k], -mq) - xh * mx));
        }
        st_pack<TX, VEC>(o + c, v);
      }
    }
    cx = nx;
    cg = ng;
  }
  pdl_launch_dependents();
  // the CTA's partial of dw (and db)
  float* part = p.part + (size_t)blockIdx.x * 2 * d;
  if constexpr (WARP) {
    const int row = threadIdx.x >> 5;
    for (int k = 0; k < rpc; ++k) {   // warps add in order
      if (row == k)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          float* a = comb + e * 32 + t;
          *a = k ? *a + dw[e] : dw[e];
          if constexpr (!RMS) a[E * 32] = k ? a[E * 32] + db[e] : db[e];
        }
      __syncthreads();
    }
    if (row != 0) return;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      dw[e] = comb[e * 32 + t];
      if constexpr (!RMS) db[e] = comb[(E + e) * 32 + t];
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int c = ((e / VEC) * tpr + t) * VEC + e % VEC;
    if (c < d) {
      part[c] = dw[e];
      if constexpr (!RMS)
        if (p.db != nullptr) part[d + c] = db[e];
    }
  }
}

// out[c] = sum over the CTAs' partials: 32 columns per CTA, 32 strided sums
// each, joined in order.
__global__ void __launch_bounds__(1024) norm_reduce_kernel(const float* part, int n, int d,
                                                           float* dw, float* db) {
  __shared__ float s[32][33];
  const int cx = threadIdx.x & 31, k = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + cx;
  const int which = blockIdx.y;   // 0: dw, 1: db
  float a = 0.f;
  pdl_wait();
  if (c < d) {
    const float* q = part + (size_t)which * d + c;
#pragma unroll 4
    for (int i = k; i < n; i += 32) a += q[(size_t)i * 2 * d];
  }
  s[k][cx] = a;
  __syncthreads();
  // warp k joins column k
  float v = s[cx][k];
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  const int cc = blockIdx.x * 32 + k;
  if (cx == 0 && cc < d) (which ? db : dw)[cc] = v;
}

// Threads of a row's CTA (0: a warp per row).
int norm_threads(int d) {
  if (d <= 256) return 0;
  const int per = d <= 8192 ? 8 : 32;
  return (d + 32 * per - 1) / (32 * per) * 32;
}
// CTAs per SM of the persistent grids: 768 threads, as many as 80 registers per
// thread allow (one CTA where a thread holds 32 elements or has 64 registers).
int norm_per_sm(int d, int nt) { return d > 8192 || nt > 768 ? 1 : 768 / nt; }

// vec: widest vector (8 when both sides are bf16, else 4) that the row starts
// and lengths allow, else single elements.
int norm_vec(int d, int dtype_x, int dtype_y, bool ok8, bool ok4) {
  if (dtype_x == M3_BF16 && dtype_y == M3_BF16 && ok8 && d % 8 == 0) return 8;
  return ok4 && d % 4 == 0 ? 4 : 1;
}

// The instantiation of a row length: f<VEC, NV, WARP, MAXT, MINB>(threads, grid).
template <int E, typename F>
cudaError_t norm_size(int vec, int nt, F&& f) {
  auto with = [&](auto v) -> cudaError_t {
    constexpr int VEC = decltype(v)::value, NV = E / VEC;
    if constexpr (E == 8)
      if (nt == 0) return f.template operator()<VEC, NV, true, 128, 6>(128);
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
// Forward rows a warp holds at E elements per lane.
template <int E, typename F>
cudaError_t norm_warp(int vec, F&& f) {
  constexpr int MINB = E <= 16 ? 5 : 4;
  if constexpr (std::decay_t<F>::kWide)
    if (vec == 8) return f.template operator()<8, E / 8, true, 128, MINB>(128);
  return vec == 4 ? f.template operator()<4, E / 4, true, 128, MINB>(128)
                  : f.template operator()<1, E, true, 128, MINB>(128);
}
template <typename F>
cudaError_t norm_dispatch(int d, int vec, F&& f) {
  const int nt = norm_threads(d);
  if constexpr (std::decay_t<F>::kWarpRows) {
    if (d > 256 && d <= 512) return norm_warp<16>(vec, f);
    if (d > 512 && d <= 768) return norm_warp<24>(vec, f);
    if (d > 768 && d <= 1024) return norm_warp<32>(vec, f);
  }
  return d <= 8192 ? norm_size<8>(vec, nt, f) : norm_size<32>(vec, nt, f);
}

template <typename TX, typename TY>
struct LaunchFwd {
  static constexpr bool kWide = sizeof(TX) == 2 && sizeof(TY) == 2, kWarpRows = true;
  const NormParams& p;
  cudaStream_t s;
  template <int VEC, int NV, bool WARP, int MAXT, int MINB>
  cudaError_t operator()(int nt) {
    const int rpc = WARP ? MAXT / 32 : 1;
    const long long want = (p.rows + rpc - 1) / rpc;
    const long long cap = (long long)p.sms * (WARP ? MINB : norm_per_sm(p.d, nt));
    const int grid = (int)(want < cap ? want : cap);
    if (p.rms) norm_fwd_kernel<TX, TY, VEC, NV, WARP, MAXT, MINB, true><<<grid, nt, 0, s>>>(p);
    else norm_fwd_kernel<TX, TY, VEC, NV, WARP, MAXT, MINB, false><<<grid, nt, 0, s>>>(p);
    return cudaGetLastError();
  }
};

template <typename TX, typename TY>
struct LaunchBwd {
  static constexpr bool kWide = sizeof(TX) == 2 && sizeof(TY) == 2, kWarpRows = false;
  const NormBwdParams& p;
  cudaStream_t s;
  template <int VEC, int NV, bool WARP, int MAXT, int MINB>
  cudaError_t operator()(int nt) {
    const int ctas = norm_bwd_ctas(p.rows, p.d, p.sms);
    if (p.rms) norm_bwd_kernel<TX, TY, VEC, NV, WARP, MAXT, MINB, true><<<ctas, nt, 0, s>>>(p);
    else norm_bwd_kernel<TX, TY, VEC, NV, WARP, MAXT, MINB, false><<<ctas, nt, 0, s>>>(p);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    return launch_maybe_pdl(true, norm_reduce_kernel,
                            dim3((p.d + 31) / 32, p.db != nullptr ? 2 : 1), dim3(1024), 0, s,
                            (const float*)p.part, ctas, p.d, p.dw, p.db);
  }
};

}  // namespace

int norm_bwd_ctas(long long rows, int d, int sms) {
  const int nt = norm_threads(d), rpc = nt ? 1 : 4;
  const long long want = (rows + rpc - 1) / rpc, cap = (long long)sms * norm_per_sm(d, nt ? nt : 128);
  return (int)(want < cap ? want : cap);
}

cudaError_t launch_norm_fwd(const NormParams& p, cudaStream_t s) {
  const int ex = dsize(p.dtype_x), ey = dsize(p.dtype_y);
  const int vec = norm_vec(p.d, p.dtype_x, p.dtype_y,
                           aligned(p.x, 16) && aligned(p.y, 16) && p.ld_x % 8 == 0,
                           aligned(p.x, 4 * ex) && aligned(p.y, 4 * ey) && p.ld_x % 4 == 0);
  const bool xb = p.dtype_x == M3_BF16, yb = p.dtype_y == M3_BF16;
  if (xb && yb) return norm_dispatch(p.d, vec, LaunchFwd<__nv_bfloat16, __nv_bfloat16>{p, s});
  if (xb) return norm_dispatch(p.d, vec, LaunchFwd<__nv_bfloat16, float>{p, s});
  if (yb) return norm_dispatch(p.d, vec, LaunchFwd<float, __nv_bfloat16>{p, s});
  return norm_dispatch(p.d, vec, LaunchFwd<float, float>{p, s});
}

cudaError_t launch_norm_bwd(const NormBwdParams& p, cudaStream_t s) {
  const int ex = dsize(p.dtype_x), ey = dsize(p.dtype_y);
  const int vec = norm_vec(
      p.d, p.dtype_x, p.dtype_y,
      aligned(p.x, 16) && aligned(p.g, 16) && aligned(p.dx, 16) && p.ld_x % 8 == 0,
      aligned(p.x, 4 * ex) && aligned(p.g, 4 * ey) && aligned(p.dx, 4 * ex) && p.ld_x % 4 == 0);
  const bool xb = p.dtype_x == M3_BF16, yb = p.dtype_y == M3_BF16;
  if (xb && yb) return norm_dispatch(p.d, vec, LaunchBwd<__nv_bfloat16, __nv_bfloat16>{p, s});
  if (xb) return norm_dispatch(p.d, vec, LaunchBwd<__nv_bfloat16, float>{p, s});
  if (yb) return norm_dispatch(p.d, vec, LaunchBwd<float, __nv_bfloat16>{p, s});
  return norm_dispatch(p.d, vec, LaunchBwd<float, float>{p, s});
}

}  // namespace m3
