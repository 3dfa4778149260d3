// Layer norm and RMS norm over rows of d elements, forward and backward.
//
//   mu = mean(x) (0 for RMS), v = mean((x - mu)^2), r = 1 / sqrt(v + eps)
//   xh = (x - mu) r,  y = xh w + b
//   with q = g w:  dx = r (q - mean(q) - xh mean(q xh))   (RMS: no mean(q))
//                  dw = sum over rows of g xh,  db = sum over rows of g
//
// Bound by memory: forward reads x and writes y, backward reads x and g and
// writes dx.  So every row is read once and stays in registers between the
// statistics and the output: TPR threads hold one row (a warp up to 1024
// elements, else 128, 512 or 1024 threads), at most 32 elements each; the
// variance is taken from the centred values in registers (no cancellation of
// mean(x^2) - mu^2).  The grid is persistent: weights stay in registers over a
// CTA's rows, the next row's loads are issued before the present row is
// reduced, and the backward keeps the weight gradients of its columns in
// registers over all its rows.  Each CTA writes one partial row of dw (and
// db); a second launch adds the partials in a fixed order, so results do not
// depend on scheduling.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "m3_api_util.h"
#include "m3_ops.h"
#include "m3_vec.cuh"

namespace m3 {
namespace {

// Sum of N values over the TPR threads of a row (every thread gets the totals).
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* red) {
#pragma unroll
  for (int m = 16; m > 0; m >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], m);
  if constexpr (TPR > 32) {
    constexpr int W = TPR / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) red[i * W + warp] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) s += red[i * W + w];
      v[i] = s;
    }
    __syncthreads();   // red may be written again
  }
}

template <typename T, int VEC, int NV, int TPR>
struct Row {
  Pack<T, VEC> p[NV];
  __device__ __forceinline__ void load(const T* row, int d, int t) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * VEC;
      p[i] = c < d ? ld_pack<T, VEC>(row + c) : zero_pack<T, VEC>();
    }
  }
  __device__ __forceinline__ float get(int k) const { return p[k / VEC].get(k % VEC); }
};

template <int VEC, int NV, int TPR>
__device__ __forceinline__ void load_f32(float (&w)[VEC * NV], const float* src, int d, int t) {
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int c = (i * TPR + t) * VEC + j;
      w[i * VEC + j] = (src != nullptr && c < d) ? src[c] : 0.f;
    }
}

constexpr int cta_threads(int tpr) { return tpr < 128 ? 128 : tpr; }

template <typename TX, typename TY, int VEC, int NV, int TPR>
__global__ void __launch_bounds__(cta_threads(TPR)) norm_fwd_kernel(const NormParams p) {
  constexpr int E = VEC * NV, RPC = cta_threads(TPR) / TPR;
  __shared__ float red[TPR / 32 + 1];
  const int t = threadIdx.x % TPR, d = p.d;
  const TX* x = static_cast<const TX*>(p.x);
  TY* y = static_cast<TY*>(p.y);
  float w[E], b[E];
  load_f32<VEC, NV, TPR>(w, p.w, d, t);
  load_f32<VEC, NV, TPR>(b, p.b, d, t);
  const float inv_d = 1.f / (float)d;
  const long long step = (long long)gridDim.x * RPC;
  long long r = (long long)blockIdx.x * RPC + threadIdx.x / TPR;
  Row<TX, VEC, NV, TPR> cur;
  if (r < p.rows) cur.load(x + (size_t)r * p.ld_x, d, t);
  for (; r < p.rows; r += step) {
    Row<TX, VEC, NV, TPR> next;
    if (r + step < p.rows) next.load(x + (size_t)(r + step) * p.ld_x, d, t);
    float v[E];
#pragma unroll
    for (int k = 0; k < E; ++k) v[k] = cur.get(k);
    float mu = 0.f;
    if (!p.rms) {
      float s[1] = {0.f};
#pragma unroll
      for (int k = 0; k < E; ++k) s[0] += v[k];
      row_sum<TPR>(s, red);
      mu = s[0] * inv_d;
#pragma unroll
      for (int i = 0; i < NV; ++i)   // columns past d stay zero
        if ((i * TPR + t) * VEC < d)
#pragma unroll
          for (int j = 0; j < VEC; ++j) v[i * VEC + j] -= mu;
    }
    float q[1] = {0.f};
#pragma unroll
    for (int k = 0; k < E; ++k) q[0] = fmaf(v[k], v[k], q[0]);
    row_sum<TPR>(q, red);
    const float rs = rsqrtf(q[0] * inv_d + p.eps);
    if (t == 0 && p.rstd != nullptr) {
      p.rstd[r] = rs;
      if (p.mean != nullptr) p.mean[r] = mu;
    }
    TY* yr = y + (size_t)r * d;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * VEC;
      if (c < d) {
        Pack<TY, VEC> o;
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          o.put(j, fmaf(v[i * VEC + j] * rs, w[i * VEC + j], b[i * VEC + j]));
        st_pack<TY, VEC>(yr + c, o);
      }
    }
    cur = next;
  }
}

template <typename TX, typename TY, int VEC, int NV, int TPR>
__global__ void __launch_bounds__(cta_threads(TPR)) norm_bwd_kernel(const NormBwdParams p) {
  constexpr int E = VEC * NV, RPC = cta_threads(TPR) / TPR;
  __shared__ float red[2 * (TPR / 32) + 2];
  extern __shared__ float comb[];   // RPC > 1: the CTA's rows' partials meet here
  const int t = threadIdx.x % TPR, d = p.d;
  const TX* x = static_cast<const TX*>(p.x);
  const TY* g = static_cast<const TY*>(p.g);
  TX* dx = static_cast<TX*>(p.dx);
  float w[E], dw[E], db[E];
  load_f32<VEC, NV, TPR>(w, p.w, d, t);
#pragma unroll
  for (int k = 0; k < E; ++k) dw[k] = db[k] = 0.f;
  const float inv_d = 1.f / (float)d;
  const long long step = (long long)gridDim.x * RPC;
  long long r = (long long)blockIdx.x * RPC + threadIdx.x / TPR;
  Row<TX, VEC, NV, TPR> cx;
  Row<TY, VEC, NV, TPR> cg;
  if (r < p.rows) {
    cx.load(x + (size_t)r * p.ld_x, d, t);
    cg.load(g + (size_t)r * d, d, t);
  }
  for (; r < p.rows; r += step) {
    Row<TX, VEC, NV, TPR> nx;
    Row<TY, VEC, NV, TPR> ng;
    if (r + step < p.rows) {
      nx.load(x + (size_t)(r + step) * p.ld_x, d, t);
      ng.load(g + (size_t)(r + step) * d, d, t);
    }
    const float rs = p.rstd[r], mu = p.rms ? 0.f : p.mean[r];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < E; ++k) {
      // a column past d has g = 0 and w = 0, so nothing of it is counted
      const float xh = (cx.get(k) - mu) * rs, gk = cg.get(k), q = gk * w[k];
      s[0] += q;
      s[1] = fmaf(q, xh, s[1]);
      dw[k] = fmaf(gk, xh, dw[k]);
      db[k] += gk;
    }
    row_sum<TPR>(s, red);
    const float mq = p.rms ? 0.f : s[0] * inv_d, mx = s[1] * inv_d;
    TX* o = dx + (size_t)r * d;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * VEC;
      if (c < d) {
        Pack<TX, VEC> v;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const int k = i * VEC + j;
          const float xh = (cx.get(k) - mu) * rs;
          v.put(j, rs * (cg.get(k) * w[k] - mq - xh * mx));
        }
        st_pack<TX, VEC>(o + c, v);
      }
    }
    cx = nx;
    cg = ng;
  }
  // the CTA's partial of dw (and db)
  float* part = p.part + (size_t)blockIdx.x * 2 * d;
  if constexpr (RPC > 1) {
    const int row = threadIdx.x / TPR;
    for (int k = 0; k < RPC; ++k) {   // rows add in order
      if (row == k)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          float* a = comb + e * TPR + t;
          float* bb = a + E * TPR;
          *a = k ? *a + dw[e] : dw[e];
          *bb = k ? *bb + db[e] : db[e];
        }
      __syncthreads();
    }
    if (row == 0)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        dw[e] = comb[e * TPR + t];
        db[e] = comb[(E + e) * TPR + t];
      }
    else return;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int c = ((e / VEC) * TPR + t) * VEC + e % VEC;
    if (c < d) {
      part[c] = dw[e];
      if (p.db != nullptr) part[d + c] = db[e];
    }
  }
}

// out[c] = sum over the CTAs' partials: 32 columns per CTA, 8 strided sums
// each, joined in order.
__global__ void __launch_bounds__(256) norm_reduce_kernel(const float* part, int n, int d,
                                                          float* dw, float* db) {
  __shared__ float s[8][33];
  const int cx = threadIdx.x & 31, k = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + cx;
  const int which = blockIdx.y;   // 0: dw, 1: db
  float a = 0.f;
  if (c < d) {
    const float* q = part + (size_t)which * d + c;
    float a1 = 0.f, a2 = 0.f, a3 = 0.f;
    int i = k;
    for (; i + 24 < n; i += 32) {
      a += q[(size_t)i * 2 * d];
      a1 += q[(size_t)(i + 8) * 2 * d];
      a2 += q[(size_t)(i + 16) * 2 * d];
      a3 += q[(size_t)(i + 24) * 2 * d];
    }
    for (; i < n; i += 8) a += q[(size_t)i * 2 * d];
    a = (a + a1) + (a2 + a3);
  }
  s[k][cx] = a;
  __syncthreads();
  if (k == 0 && c < d) {
    float v = s[0][cx];
#pragma unroll
    for (int j = 1; j < 8; ++j) v += s[j][cx];
    (which ? db : dw)[c] = v;
  }
}

struct Plan { int tpr, nv, vec; };

// The fewest threads per row that hold it at 32 elements each.
int norm_tpr(int d) { return d <= 1024 ? 32 : d <= 4096 ? 128 : d <= 16384 ? 512 : 1024; }

// vec: widest vector (8 when both sides are bf16, else 4) that the row starts
// and lengths allow, else single elements.
int norm_vec(int d, int dtype_x, int dtype_y, bool ok8, bool ok4) {
  if (dtype_x == M3_BF16 && dtype_y == M3_BF16 && ok8 && d % 8 == 0) return 8;
  return ok4 && d % 4 == 0 ? 4 : 1;
}

// The instantiation for a row: past a warp per row, d is over a quarter (past
// 512 threads: a half) of what the row's threads hold, so only the larger
// element counts exist there.
template <int TPR, bool WIDE, typename F>
cudaError_t norm_pick(int vec, int nv, F&& f) {
  if constexpr (WIDE) {
    if (vec == 8) {
      if constexpr (TPR == 32) {
        if (nv <= 1) return f.template operator()<8, 1, TPR>();
      }
      if constexpr (TPR < 1024) {
        if (nv <= 2) return f.template operator()<8, 2, TPR>();
      }
      if (nv <= 3) return f.template operator()<8, 3, TPR>();
      return f.template operator()<8, 4, TPR>();
    }
  }
  if (vec == 4) {
    if constexpr (TPR == 32) {
      if (nv <= 2) return f.template operator()<4, 2, TPR>();
    }
    if constexpr (TPR < 1024) {
      if (nv <= 4) return f.template operator()<4, 4, TPR>();
    }
    if (nv <= 6) return f.template operator()<4, 6, TPR>();
    return f.template operator()<4, 8, TPR>();
  }
  if constexpr (TPR == 32) {
    if (nv <= 8) return f.template operator()<1, 8, TPR>();
  }
  return f.template operator()<1, 32, TPR>();
}

template <bool WIDE, typename P, typename F>
cudaError_t norm_dispatch(const P& p, F&& f) {
  const int tpr = norm_tpr(p.d);
  const int nv = (p.d + tpr * p.vec - 1) / (tpr * p.vec);
  switch (tpr) {
    case 32: return norm_pick<32, WIDE>(p.vec, nv, f);
    case 128: return norm_pick<128, WIDE>(p.vec, nv, f);
    case 512: return norm_pick<512, WIDE>(p.vec, nv, f);
    default: return norm_pick<1024, WIDE>(p.vec, nv, f);
  }
}

template <typename TX, typename TY>
struct LaunchFwd {
  const NormParams& p;
  cudaStream_t s;
  template <int VEC, int NV, int TPR>
  cudaError_t operator()() {
    constexpr int nt = cta_threads(TPR), rpc = nt / TPR;
    const long long want = (p.rows + rpc - 1) / rpc, cap = (long long)p.sms * (2048 / nt);
    const int grid = (int)(want < cap ? want : cap);
    norm_fwd_kernel<TX, TY, VEC, NV, TPR><<<grid, nt, 0, s>>>(p);
    return cudaGetLastError();
  }
};

template <typename TX, typename TY>
struct LaunchBwd {
  const NormBwdParams& p;
  cudaStream_t s;
  template <int VEC, int NV, int TPR>
  cudaError_t operator()() {
    constexpr int nt = cta_threads(TPR), rpc = nt / TPR;
    const int smem = rpc > 1 ? 2 * VEC * NV * TPR * 4 : 0;
    norm_bwd_kernel<TX, TY, VEC, NV, TPR><<<p.ctas, nt, smem, s>>>(p);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    norm_reduce_kernel<<<dim3((p.d + 31) / 32, p.db != nullptr ? 2 : 1), 256, 0, s>>>(
        p.part, p.ctas, p.d, p.dw, p.db);
    return cudaGetLastError();
  }
};

}  // namespace

int norm_bwd_ctas(long long rows, int d, int sms) {
  const int nt = cta_threads(norm_tpr(d)), rpc = nt / norm_tpr(d);
  const long long want = (rows + rpc - 1) / rpc, cap = (long long)sms * (nt >= 512 ? 1 : 4);
  return (int)(want < cap ? want : cap);
}

cudaError_t launch_norm_fwd(const NormParams& p0, cudaStream_t s) {
  NormParams p = p0;
  const int ex = dsize(p.dtype_x), ey = dsize(p.dtype_y);
  p.vec = norm_vec(p.d, p.dtype_x, p.dtype_y,
                   aligned(p.x, 16) && aligned(p.y, 16) && p.ld_x % 8 == 0,
                   aligned(p.x, 4 * ex) && aligned(p.y, 4 * ey) && p.ld_x % 4 == 0);
  const bool xb = p.dtype_x == M3_BF16, yb = p.dtype_y == M3_BF16;
  if (xb && yb) return norm_dispatch<true>(p, LaunchFwd<__nv_bfloat16, __nv_bfloat16>{p, s});
  if (xb) return norm_dispatch<false>(p, LaunchFwd<__nv_bfloat16, float>{p, s});
  if (yb) return norm_dispatch<false>(p, LaunchFwd<float, __nv_bfloat16>{p, s});
  return norm_dispatch<false>(p, LaunchFwd<float, float>{p, s});
}

cudaError_t launch_norm_bwd(const NormBwdParams& p0, cudaStream_t s) {
  NormBwdParams p = p0;
  const int ex = dsize(p.dtype_x), ey = dsize(p.dtype_y);
  p.vec = norm_vec(p.d, p.dtype_x, p.dtype_y,
                   aligned(p.x, 16) && aligned(p.g, 16) && aligned(p.dx, 16) && p.ld_x % 8 == 0,
                   aligned(p.x, 4 * ex) && aligned(p.g, 4 * ey) && aligned(p.dx, 4 * ex) &&
                       p.ld_x % 4 == 0);
  const bool xb = p.dtype_x == M3_BF16, yb = p.dtype_y == M3_BF16;
  if (xb && yb) return norm_dispatch<true>(p, LaunchBwd<__nv_bfloat16, __nv_bfloat16>{p, s});
  if (xb) return norm_dispatch<false>(p, LaunchBwd<__nv_bfloat16, float>{p, s});
  if (yb) return norm_dispatch<false>(p, LaunchBwd<float, __nv_bfloat16>{p, s});
  return norm_dispatch<false>(p, LaunchBwd<float, float>{p, s});
}

}  // namespace m3
