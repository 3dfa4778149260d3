// Short causal convolution over time, one filter of K taps per channel, with
// an optional silu: prompts (forward and backward) and single tokens.
//
//   p_t = b + sum_k w_k x_{t-K+1+k},   y_t = silu(p_t) or p_t
//   g_t = dy_t silu'(p_t),  dx_t = sum_k w_k g_{t+K-1-k},
//   dw_k = sum over b, t of g_t x_{t-K+1+k},  db = sum of g_t
//
// Rows before the sequence come from the state (the last K-1 input rows of an
// earlier part), or are zero; steps at or past a row's length have y = 0 and
// take no part in any gradient, and the new state ends at the length.
//
// Bound by memory forward (x in, y out) and by instructions backward (x and dy
// in, dx out, and silu' of every element: about 45 per element at first, a third
// of them moves of the windows).  A thread owns a vector of channels and a run of
// TT steps and keeps the K rows of the filter's window in registers, so each row
// is loaded once plus K-1 halo rows per run (L1/L2 hits: the neighbouring run
// loads the same lines); the next group of rows is in flight while the present
// one is computed on.  Products are packed pairs of channels.  The backward
// recomputes p from x rather than storing it.  Weight gradients stay in registers
// over all runs of a thread; a CTA joins its 8 workers per channel in order and
// writes one partial, and a second launch adds the partials in a fixed order.
// 512 rows x 64 steps x 1536 channels, K = 4, bf16: 47 us forward (4.3 TB/s),
// 84 us backward (3.6 TB/s); 60 and 186 us at first.  In fp32: 66 us forward (6.1
// TB/s), 222 us backward (2.7 TB/s), whose filter of four taps does not fit the 128
// registers of two CTAs per SM (424 bytes per thread in local memory).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "m3_api_util.h"
#include "m3_math.cuh"
#include "m3_ops.h"
#include "m3_pdl.cuh"
#include "m3_vec.cuh"

namespace m3 {
namespace {

constexpr int kAhead = 4;      // rows in flight per thread (backward: of x and dy, twice)
constexpr int kAheadFwd = 8;

// V fp32 values as packed pairs (V = 1: the second half idles).
template <int V> struct Vals {
  static constexpr int H = (V + 1) / 2;
  float2 v[H];
  __device__ __forceinline__ float get(int j) const { return j & 1 ? v[j / 2].y : v[j / 2].x; }
  __device__ __forceinline__ void set(float a) {
#pragma unroll
    for (int i = 0; i < H; ++i) v[i] = f2(a);
  }
  template <typename T>
  __device__ __forceinline__ void from(const Pack<T, V>& p) {
#pragma unroll
    for (int i = 0; i < H; ++i) v[i] = make_float2(p.get(2 * i), V > 1 ? p.get(2 * i + 1) : 0.f);
  }
  // this += a * b
  __device__ __forceinline__ void fma(const Vals& a, const Vals& b) {
#pragma unroll
    for (int i = 0; i < H; ++i) v[i] = __ffma2_rn(a.v[i], b.v[i], v[i]);
  }
};

__device__ __forceinline__ int row_length(const int* lengths, int b, int L) {
  if (lengths == nullptr) return L;
  const int n = lengths[b];
  return n < 0 ? 0 : n > L ? L : n;
}

// Input row t of sequence b as fp32 (t < 0: the state's rows, or zeros).
template <typename T, int V>
struct Rows {
  const T* x; const T* state;   // already at the channel
  long long ld; int D, K;
  __device__ __forceinline__ Pack<T, V> at(int t) const {
    if (t >= 0) return ld_pack<T, V>(x + (size_t)t * ld);
    if (state != nullptr) return ld_pack<T, V>(state + (size_t)(t + K - 1) * D);
    return zero_pack<T, V>();
  }
};

template <int V, int K>
__device__ __forceinline__ void load_filter(Vals<V> (&w)[K], Vals<V>& b, const float* pw,
                                            const float* pb, int c) {
  alignas(16) float t[K + 1][2 * Vals<V>::H] = {};
  // the taps of V channels are V * K neighbours
  if constexpr (V == 4) {
    alignas(16) float f[V * K];
#pragma unroll
    for (int i = 0; i < K; ++i)
      *reinterpret_cast<float4*>(f + 4 * i) = reinterpret_cast<const float4*>(pw + (size_t)c * K)[i];
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int k = 0; k < K; ++k) t[k][j] = f[j * K + k];
    if (pb != nullptr)
      *reinterpret_cast<float4*>(t[K]) = *reinterpret_cast<const float4*>(pb + c);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
#pragma unroll
      for (int k = 0; k < K; ++k) t[k][j] = pw[(size_t)(c + j) * K + k];
      t[K][j] = pb != nullptr ? pb[c + j] : 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < Vals<V>::H; ++i) {
#pragma unroll
    for (int k = 0; k < K; ++k) w[k].v[i] = make_float2(t[k][2 * i], t[k][2 * i + 1]);
    b.v[i] = make_float2(t[K][2 * i], t[K][2 * i + 1]);
  }
}

template <typename T, int V, int K>
__global__ void __launch_bounds__(128) conv_fwd_kernel(const ConvParams p) {
  const int lanes = p.D / V, runs = (p.L + p.tt - 1) / p.tt;
  const long long idx = (long long)blockIdx.x * 128 + threadIdx.x;
  if (idx >= (long long)lanes * runs * p.B) return;
  const int c = (int)(idx % lanes) * V;
  const long long q = idx / lanes;
  const int run = (int)(q % runs), b = (int)(q / runs);
  const int n = row_length(p.lengths, b, p.L);
  Rows<T, V> in{static_cast<const T*>(p.x) + (size_t)b * p.L * p.ld_x + c,
                p.state ? static_cast<const T*>(p.state) + (size_t)b * (K - 1) * p.D + c : nullptr,
                p.ld_x, p.D, K};
  if (run == 0 && p.state_out != nullptr) {
    T* so = static_cast<T*>(p.state_out) + (size_t)b * (K - 1) * p.D + c;
#pragma unroll
    for (int j = 0; j < K - 1; ++j) st_pack<T, V>(so + (size_t)j * p.D, in.at(n - (K - 1) + j));
  }
  const int t0 = run * p.tt, t1 = min(t0 + p.tt, p.L), te = min(t1, n);
  T* y = static_cast<T*>(p.y) + (size_t)b * p.L * p.D + c;
  int t = t0;
  if (t < te) {
    Vals<V> w[K], bias, win[K];
    load_filter<V, K>(w, bias, p.w, p.b, c);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) win[k + 1].from(in.at(t0 - (K - 1) + k));
    auto one = [&](const Pack<T, V>& r, int tt) {
#pragma unroll
      for (int k = 0; k < K - 1; ++k) win[k] = win[k + 1];
      win[K - 1].from(r);
      Vals<V> a = bias;
#pragma unroll
      for (int k = 0; k < K; ++k) a.fma(w[k], win[k]);
      Pack<T, V> o;
#pragma unroll
      for (int j = 0; j < V; ++j) o.put(j, p.silu ? silu_f(a.get(j)) : a.get(j));
      st_pack<T, V>(y + (size_t)tt * p.D, o);
    };
    // two groups of rows in flight: one computed on, one being loaded
    Pack<T, V> r[kAheadFwd], next[kAheadFwd];
    auto fetch = [&](Pack<T, V> (&q)[kAheadFwd], int at) {
      const T* px = in.x + (size_t)at * in.ld;
#pragma unroll
      for (int i = 0; i < kAheadFwd; ++i) q[i] = ld_pack<T, V>(px + i * in.ld);
    };
    if (t + kAheadFwd <= te) fetch(r, t);
    for (; t + kAheadFwd <= te; t += kAheadFwd) {
      if (t + 2 * kAheadFwd <= te) fetch(next, t + kAheadFwd);
#pragma unroll
      for (int i = 0; i < kAheadFwd; ++i) one(r[i], t + i);
#pragma unroll
      for (int i = 0; i < kAheadFwd; ++i) r[i] = next[i];
    }
    for (; t < te; ++t) one(ld_pack<T, V>(in.x + (size_t)t * in.ld), t);
  }
  for (; t < t1; ++t) st_pack<T, V>(y + (size_t)t * p.D, zero_pack<T, V>());
}

constexpr int kWorkers = 8;    // workers (warps) per CTA of the backward

template <typename T, int V, int K>
__global__ void __launch_bounds__(32 * kWorkers, K <= 4 ? 2 : 1) conv_bwd_kernel(const ConvBwdParams p) {
  __shared__ float comb[K + 1][32 * V];
  const int lane = threadIdx.x & 31, wk = threadIdx.x >> 5;
  const int c = (blockIdx.x * 32 + lane) * V;
  const bool live = c < p.D;
  const int runs = (p.L + p.tt - 1) / p.tt;
  const long long tasks = (long long)runs * p.B;
  Vals<V> dw[K], db;
  db.set(0.f);
#pragma unroll
  for (int k = 0; k < K; ++k) dw[k].set(0.f);
  if (live) {
    Vals<V> w[K], bias;
    load_filter<V, K>(w, bias, p.w, p.b, c);
    for (long long q = (long long)blockIdx.y * kWorkers + wk; q < tasks;
         q += (long long)gridDim.y * kWorkers) {
      const int run = (int)(q % runs), b = (int)(q / runs);
      const int n = row_length(p.lengths, b, p.L);
      Rows<T, V> in{
          static_cast<const T*>(p.x) + (size_t)b * p.L * p.ld_x + c,
          p.state ? static_cast<const T*>(p.state) + (size_t)b * (K - 1) * p.D + c : nullptr,
          p.ld_x, p.D, K};
      const T* g = static_cast<const T*>(p.g) + (size_t)b * p.L * p.D + c;
      T* dx = static_cast<T*>(p.dx) + (size_t)b * p.L * p.D + c;
      const int t0 = run * p.tt, t1 = min(t0 + p.tt, p.L), te = min(t1, n);
      // steps [t0, tg) are read: K-1 past the run, for its last dx rows
      const int tg = te > t0 ? min(te + K - 1, n) : t0;
      Pack<T, V> rx[kAhead], rg[kAhead];
      auto fetch = [&](int t) {
        const T* px = in.x + (size_t)t * in.ld;
        const T* pg = g + (size_t)t * p.D;
        if (t + kAhead <= tg) {
#pragma unroll
          for (int i = 0; i < kAhead; ++i) {
            rx[i] = ld_pack<T, V>(px + i * in.ld);
            rg[i] = ld_pack<T, V>(pg + (size_t)i * p.D);
          }
        } else {
#pragma unroll
          for (int i = 0; i < kAhead; ++i)
            if (t + i < tg) {
              rx[i] = ld_pack<T, V>(px + i * in.ld);
              rg[i] = ld_pack<T, V>(pg + (size_t)i * p.D);
            }
        }
      };
      fetch(t0);
      Vals<V> win[K], gw[K];
#pragma unroll
      for (int k = 0; k < K; ++k) gw[k].set(0.f);
      if (te > t0) {
#pragma unroll
        for (int k = 0; k < K - 1; ++k) win[k + 1].from(in.at(t0 - (K - 1) + k));
      }
      // after step t the window of g holds g[t-K+1 .. t]: dx[t-K+1] is complete
      auto emit = [&](int s) {
        Vals<V> a;
        a.set(0.f);
#pragma unroll
        for (int k = 0; k < K; ++k) a.fma(w[k], gw[K - 1 - k]);
        Pack<T, V> o;
#pragma unroll
        for (int j = 0; j < V; ++j) o.put(j, a.get(j));
        st_pack<T, V>(dx + (size_t)s * p.D, o);
      };
      // One step; WHOLE: inside the run, with a dx row to write (no conditions, so
      // that the windows of a group of steps are renamed instead of moved).
      auto step = [&](auto whole, const Pack<T, V>& px, const Pack<T, V>& pg, int t) {
        constexpr bool WHOLE = decltype(whole)::value;
#pragma unroll
        for (int k = 0; k < K - 1; ++k) {
          win[k] = win[k + 1];
          gw[k] = gw[k + 1];
        }
        win[K - 1].from(px);
        Vals<V> gt;
        gt.from(pg);
        if (p.silu) {
          Vals<V> a = bias;
#pragma unroll
          for (int k = 0; k < K; ++k) a.fma(w[k], win[k]);
#pragma unroll
          for (int h = 0; h < Vals<V>::H; ++h) {
            gt.v[h].x *= dsilu_f(a.v[h].x, sigmoid_f(a.v[h].x));
            if (V > 1) gt.v[h].y *= dsilu_f(a.v[h].y, sigmoid_f(a.v[h].y));
          }
        }
        gw[K - 1] = gt;
        if (WHOLE || t < te) {   // halo steps belong to the next run
#pragma unroll
          for (int h = 0; h < Vals<V>::H; ++h) db.v[h] = __fadd2_rn(db.v[h], gt.v[h]);
#pragma unroll
          for (int k = 0; k < K; ++k) dw[k].fma(gt, win[k]);
        }
        if (WHOLE || t - (K - 1) >= t0) emit(t - (K - 1));
      };
      for (int tb = t0; tb < tg; tb += kAhead) {
        Pack<T, V> cx[kAhead], cg[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          cx[i] = rx[i];
          cg[i] = rg[i];
        }
        fetch(tb + kAhead);
        if (tb - (K - 1) >= t0 && tb + kAhead <= te) {
#pragma unroll
          for (int i = 0; i < kAhead; ++i) step(std::true_type(), cx[i], cg[i], tb + i);
        } else {
#pragma unroll
          for (int i = 0; i < kAhead; ++i)
            if (tb + i < tg) step(std::false_type(), cx[i], cg[i], tb + i);
        }
      }
      // the sequence's end: g past it is zero
      for (int t = tg; t - (K - 1) < te; ++t) {
#pragma unroll
        for (int k = 0; k < K - 1; ++k) gw[k] = gw[k + 1];
        gw[K - 1].set(0.f);
        if (t - (K - 1) >= t0) emit(t - (K - 1));
      }
      for (int s = max(te, t0); s < t1; ++s)
        st_pack<T, V>(dx + (size_t)s * p.D, zero_pack<T, V>());
    }
  }
  pdl_launch_dependents();
  for (int k = 0; k < kWorkers; ++k) {   // workers add in order
    if (wk == k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
#pragma unroll
        for (int i = 0; i < K; ++i) {
          float* a = &comb[i][j * 32 + lane];
          *a = k ? *a + dw[i].get(j) : dw[i].get(j);
        }
        float* a = &comb[K][j * 32 + lane];
        *a = k ? *a + db.get(j) : db.get(j);
      }
    __syncthreads();
  }
  if (wk == 0 && live) {
    float* part = p.part + (size_t)blockIdx.y * (K + 1) * p.D;
#pragma unroll
    for (int i = 0; i <= K; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) part[(size_t)i * p.D + c + j] = comb[i][j * 32 + lane];
  }
}

// dw[c][k], db[c]: the partials of one (tap, channel) in a fixed order.
__global__ void __launch_bounds__(256) conv_reduce_kernel(const float* part, int n, int D, int K,
                                                          float* dw, float* db) {
  __shared__ float s[8][33];
  const int cx = threadIdx.x & 31, k = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + cx, tap = blockIdx.y;
  float a = 0.f;
  pdl_wait();
  if (c < D) {
    const float* q = part + (size_t)tap * D + c;
    for (int i = k; i < n; i += 8) a += q[(size_t)i * (K + 1) * D];
  }
  s[k][cx] = a;
  __syncthreads();
  if (k == 0 && c < D) {
    float v = s[0][cx];
#pragma unroll
    for (int j = 1; j < 8; ++j) v += s[j][cx];
    if (tap < K) dw[(size_t)c * K + tap] = v;
    else if (db != nullptr) db[c] = v;
  }
}

// One token per row: the window is [state, x]; the state moves up by one row.  A
// thread takes its channels of kStepRows rows, all loads ahead of the arithmetic.
constexpr int kStepRows = 4;

template <typename T, int V, int K>
__global__ void __launch_bounds__(128) conv_step_kernel(const ConvStepParams p) {
  const int lanes = p.D / V;
  const long long idx = (long long)blockIdx.x * 128 + threadIdx.x;
  const long long blocks = (p.B + kStepRows - 1) / kStepRows;
  if (idx >= lanes * blocks) return;
  const int c = (int)(idx % lanes) * V;
  const size_t b0 = (size_t)(idx / lanes) * kStepRows;
  const int rows = (int)min((size_t)kStepRows, (size_t)p.B - b0);
  T* st = static_cast<T*>(p.state) + b0 * (K - 1) * p.D + c;
  Pack<T, V> r[kStepRows][K];
#pragma unroll
  for (int i = 0; i < kStepRows; ++i)
    if (i < rows) {
#pragma unroll
      for (int k = 0; k < K - 1; ++k)
        r[i][k] = ld_pack<T, V>(st + ((size_t)i * (K - 1) + k) * p.D);
      r[i][K - 1] = ld_pack<T, V>(static_cast<const T*>(p.x) + (b0 + i) * p.ld_x + c);
    }
  Vals<V> w[K], bias;
  load_filter<V, K>(w, bias, p.w, p.b, c);
#pragma unroll
  for (int i = 0; i < kStepRows; ++i)
    if (i < rows) {
      Vals<V> a = bias;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        Vals<V> x;
        x.from(r[i][k]);
        a.fma(w[k], x);
      }
      Pack<T, V> o;
#pragma unroll
      for (int j = 0; j < V; ++j) o.put(j, p.silu ? silu_f(a.get(j)) : a.get(j));
#pragma unroll
      for (int k = 0; k < K - 1; ++k)
        st_pack<T, V>(st + ((size_t)i * (K - 1) + k) * p.D, r[i][k + 1]);
      st_pack<T, V>(static_cast<T*>(p.y) + (b0 + i) * p.D + c, o);
    }
}

// Calls f<T, V, K>() for an element type, vector and width.
template <typename T, int V, typename F>
cudaError_t conv_width(int K, F&& f) {
  switch (K) {
    case 1: return f.template operator()<T, V, 1>();
    case 2: return f.template operator()<T, V, 2>();
    case 3: return f.template operator()<T, V, 3>();
    case 4: return f.template operator()<T, V, 4>();
    case 5: return f.template operator()<T, V, 5>();
    case 6: return f.template operator()<T, V, 6>();
    case 7: return f.template operator()<T, V, 7>();
    default: return f.template operator()<T, V, 8>();
  }
}

template <typename F>
cudaError_t conv_dispatch(int dtype, bool vec, int K, F&& f) {
  if (dtype == M3_BF16)
    return vec ? conv_width<__nv_bfloat16, 4>(K, f) : conv_width<__nv_bfloat16, 1>(K, f);
  return vec ? conv_width<float, 4>(K, f) : conv_width<float, 1>(K, f);
}

struct FwdLaunch {
  const ConvParams& p;
  cudaStream_t s;
  template <typename T, int V, int K>
  cudaError_t operator()() {
    const long long n = (long long)(p.D / V) * ((p.L + p.tt - 1) / p.tt) * p.B;
    conv_fwd_kernel<T, V, K><<<(unsigned)((n + 127) / 128), 128, 0, s>>>(p);
    return cudaGetLastError();
  }
};

struct BwdLaunch {
  const ConvBwdParams& p;
  cudaStream_t s;
  template <typename T, int V, int K>
  cudaError_t operator()() {
    const dim3 grid((unsigned)((p.D / V + 31) / 32), (unsigned)p.workers);
    conv_bwd_kernel<T, V, K><<<grid, 32 * kWorkers, 0, s>>>(p);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    return launch_maybe_pdl(true, conv_reduce_kernel,
                            dim3((unsigned)((p.D + 31) / 32), (unsigned)(K + 1)), dim3(256), 0, s,
                            (const float*)p.part, p.workers, p.D, K, p.dw, p.db);
  }
};

struct StepLaunch {
  const ConvStepParams& p;
  cudaStream_t s;
  template <typename T, int V, int K>
  cudaError_t operator()() {
    const long long n = (long long)(p.D / V) * ((p.B + kStepRows - 1) / kStepRows);
    conv_step_kernel<T, V, K><<<(unsigned)((n + 127) / 128), 128, 0, s>>>(p);
    return cudaGetLastError();
  }
};

}  // namespace

cudaError_t launch_conv_fwd(const ConvParams& p0, cudaStream_t s) {
  ConvParams p = p0;
  const int a = 4 * dsize(p.dtype);
  const bool vec = p.D % 4 == 0 && p.ld_x % 4 == 0 && aligned(p.x, a) && aligned(p.y, a) &&
                   aligned(p.state, a) && aligned(p.state_out, a) && aligned(p.w, 16) &&
                   aligned(p.b, 16);
  // long runs read fewer halo rows, short ones give more threads
  const long long lanes = vec ? p.D / 4 : p.D;
  p.tt = 32;
  while (p.tt > 4 && lanes * p.B * ((p.L + p.tt - 1) / p.tt) < (long long)p.sms * 1024) p.tt /= 2;
  return conv_dispatch(p.dtype, vec, p.K, FwdLaunch{p, s});
}

void conv_bwd_plan(int B, int L, int D, int sms, int* workers, int* tt) {
  // channel groups of 32 lanes of 4 channels (or of 1: more groups, the same
  // partials per channel); one wave of two CTAs per SM
  const long long groups = (D + 127) / 128;
  int t = 32;
  while (t > 8 && groups * B * ((L + t - 1) / t) < (long long)sms * 2 * kWorkers) t /= 2;
  const long long tasks = (long long)B * ((L + t - 1) / t);
  long long w = (long long)sms * 2 / groups;
  const long long most = (tasks + kWorkers - 1) / kWorkers;
  if (w > most) w = most;
  if (w < 1) w = 1;
  *workers = (int)w;
  *tt = t;
}

cudaError_t launch_conv_bwd(const ConvBwdParams& p, cudaStream_t s) {
  const int a = 4 * dsize(p.dtype);
  const bool vec = p.D % 4 == 0 && p.ld_x % 4 == 0 && aligned(p.x, a) && aligned(p.g, a) &&
                   aligned(p.dx, a) && aligned(p.state, a) && aligned(p.w, 16) && aligned(p.b, 16);
  return conv_dispatch(p.dtype, vec, p.K, BwdLaunch{p, s});
}

cudaError_t launch_conv_step(const ConvStepParams& p, cudaStream_t s) {
  const int a = 4 * dsize(p.dtype);
  const bool vec = p.D % 4 == 0 && p.ld_x % 4 == 0 && aligned(p.x, a) && aligned(p.y, a) &&
                   aligned(p.state, a) && aligned(p.w, 16) && aligned(p.b, 16);
  return conv_dispatch(p.dtype, vec, p.K, StepLaunch{p, s});
}

}  // namespace m3
