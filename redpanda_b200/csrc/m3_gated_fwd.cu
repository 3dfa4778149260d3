// Gated linear recurrence, forward over whole sequences and single tokens.
// Formulas and the precision of the decay: m3_gated.cuh.
//
// A CTA holds 64 channels, two per lane, and its warps hold consecutive runs of 8
// steps; a cluster of up to 8 CTAs holds that many runs more where there are too
// few rows and channel tiles for the GPU.  Each pass of a CTA (cluster) over its
// runs loads every input once: a thread computes a and b = m i x of its steps,
// the run's product and sum, joins the runs ahead (join()), and walks its steps
// from there.  The copies of the next pass's rows are in flight meanwhile.
#include "m3_gated.cuh"

#include <type_traits>

#include "m3_api_util.h"
#include "m3_ops.h"

namespace m3 {
namespace {

__device__ __forceinline__ int row_length(const int* lengths, int b, int L) {
  if (lengths == nullptr) return L;
  const int n = lengths[b];
  return n < 0 ? 0 : n > L ? L : n;
}

template <typename T>
__global__ void __launch_bounds__(256, 3) gated_fwd_kernel(const GatedParams p) {
  extern __shared__ __align__(16) char smem[];
  __shared__ Joint joint;
  constexpr int TS = kGatedSteps;
  using St = Stage<T, 3>;
  const int lane = threadIdx.x, w = threadIdx.y, W = blockDim.y, S = p.splits;
  const int rank = blockIdx.x % S, c0 = blockIdx.x / S * kGatedTile, c = c0 + 2 * lane;
  const int left = p.D - c, D = p.D, L = p.L, span = S * W * TS;
  const int at0 = (rank * W + w) * TS;               // of this warp in a pass
  const bool vec = p.vec != 0;
  char* buf = smem + w * St::kBytes;
  St st{{static_cast<const T*>(p.x), static_cast<const T*>(p.rg), static_cast<const T*>(p.ig)},
        {p.ld_x, p.ld_r, p.ld_i}};
  const float2 dec = load_pair(p.decay + c, left);
  const float2 k = make_float2(-p.c * softplus_f(dec.x), -p.c * softplus_f(dec.y));
  int flip = 0;
  if (S > 1) cluster_sync();                         // every CTA runs before its memory is written
  for (int b = blockIdx.y; b < p.B; b += gridDim.y) {
    const int n = row_length(p.lengths, b, L);
    const long long base = (long long)b * L;
    T* y = static_cast<T*>(p.y) + (size_t)base * D + c;
    float2 carry = p.h0 != nullptr ? load_pair(p.h0 + (size_t)b * D + c, left) : f2(0.f);
    int t0 = at0;
    if (n > 0) st.issue(buf, base, t0, n, c0, D, vec);
    for (int s0 = 0; s0 < n; s0 += span, t0 += span) {
      float2 a[TS], v[TS];
      Run run{f2(1.f), f2(0.f)};
      St::wait();
#pragma unroll
      for (int i = 0; i < TS; ++i) {
        const float2 x = St::get(buf, 0, i), r = sigmoid2(St::get(buf, 1, i)),
                     g = sigmoid2(St::get(buf, 2, i));
        float2 e, m, inv;
        decay2(mul2(k, r), e, m);
        root2(m, m, inv);
        const bool live = t0 + i < n;                // else: the state stays
        a[i] = live ? e : f2(1.f);
        v[i] = live ? mul2(mul2(m, g), x) : f2(0.f);
        run.V = fma2(a[i], run.V, v[i]);
        run.P = mul2(a[i], run.P);
      }
      __syncwarp();
      if (s0 + span < n) st.issue(buf, base, t0 + span, n, c0, D, vec);
      float2 h = join(joint, flip, run, w, W, rank, S, carry);
      flip ^= 1;
      if (p.ckpt != nullptr && t0 < n)
        store_pair(p.ckpt + ((size_t)b * ((L + TS - 1) / TS) + t0 / TS) * D + c, h, left,
                   D % 2 == 0);
#pragma unroll
      for (int i = 0; i < TS; ++i) {
        h = fma2(a[i], h, v[i]);
        if (t0 + i < L) store_pair(y + (size_t)(t0 + i) * D, t0 + i < n ? h : f2(0.f), left, vec);
      }
    }
    for (; t0 - at0 < L; t0 += span)                 // steps past the length
      for (int i = 0; i < TS && t0 + i < L; ++i)
        store_pair(y + (size_t)(t0 + i) * D, f2(0.f), left, vec);
    if (p.h_last != nullptr && rank == 0 && w == 0)
      store_pair(p.h_last + (size_t)b * D + c, carry, left, false);
  }
}

// One token per row: a thread owns V channels and walks rows.
template <typename T, int V>
__global__ void __launch_bounds__(256) gated_step_kernel(const GatedStepParams p) {
  const int c = (blockIdx.x * 32 + threadIdx.x) * V;
  if (c >= p.D) return;
  float k[V];
#pragma unroll
  for (int j = 0; j < V; ++j) k[j] = -p.c * softplus_f(p.decay[c + j]);
  for (int b = blockIdx.y * blockDim.y + threadIdx.y; b < p.B; b += gridDim.y * blockDim.y) {
    const Pack<T, V> x = ld_pack<T, V>(static_cast<const T*>(p.x) + (size_t)b * p.ld_x + c),
                     r = ld_pack<T, V>(static_cast<const T*>(p.rg) + (size_t)b * p.ld_r + c),
                     g = ld_pack<T, V>(static_cast<const T*>(p.ig) + (size_t)b * p.ld_i + c);
    float* hp = p.h + (size_t)b * p.D + c;
    Pack<float, V> h = ld_pack<float, V>(hp);
    Pack<T, V> y;
    y.zero();
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      constexpr int o = V > 1 ? 1 : 0;
      float2 a, m, inv;
      decay2(mul2(make_float2(k[j], k[j + o]),
                  sigmoid2(make_float2(r.get(j), r.get(j + o)))), a, m);
      root2(m, m, inv);
      const float2 in = mul2(mul2(m, sigmoid2(make_float2(g.get(j), g.get(j + o)))),
                             make_float2(x.get(j), x.get(j + o)));
      const float2 q = fma2(a, make_float2(h.get(j), h.get(j + o)), in);
      h.put(j, q.x);
      y.put(j, q.x);
      if (V > 1) {
        h.put(j + o, q.y);
        y.put(j + o, q.y);
      }
    }
    st_pack<float, V>(hp, h);
    st_pack<T, V>(static_cast<T*>(p.y) + (size_t)b * p.D + c, y);
  }
}

template <typename T, int V>
cudaError_t step_impl(const GatedStepParams& p, cudaStream_t s) {
  const int tiles = (p.D + 32 * V - 1) / (32 * V);
  const int ty = p.B < 8 ? p.B : 8;
  long long gy = (p.B + ty - 1) / ty;
  const long long cap = (8LL * p.sms + tiles - 1) / tiles;
  if (gy > cap) gy = cap;
  if (gy > 65535) gy = 65535;
  gated_step_kernel<T, V><<<dim3(tiles, (unsigned)gy), dim3(32, ty), 0, s>>>(p);
  return cudaGetLastError();
}

template <typename T>
cudaError_t fwd_impl(const GatedParams& p, cudaStream_t s) {
  const int smem = p.warps * Stage<T, 3>::kBytes;
  const cudaError_t e = allow_smem<gated_fwd_kernel<T>>(8 * Stage<T, 3>::kBytes);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((p.D + kGatedTile - 1) / kGatedTile * p.splits), p.rows);
  cfg.blockDim = dim3(32, p.warps);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = p.splits > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, gated_fwd_kernel<T>, p);
}

}  // namespace

int gated_segments(int L) { return (L + kGatedSteps - 1) / kGatedSteps; }

void gated_plan(int B, int L, int D, int dtype, bool backward, int sms, int* warps, int* splits,
                int* rows) {
  const int per = backward ? 2 : 3;                        // CTAs per SM
  const int segs = gated_segments(L);
  *warps = segs < 8 ? segs : 8;
  const long long tiles = (D + kGatedTile - 1) / kGatedTile, wave = (long long)per * sms;
  int S = 1;
  while (S < 8 && tiles * B * S * 2 <= wave && segs >= S * 2 * *warps) S *= 2;
  *splits = S;
  long long gy = B, cap = wave / (tiles * S);
  if (cap < 1) cap = 1;
  if (cap > 65535) cap = 65535;
  if (gy > cap) {
    const long long each = (B + cap - 1) / cap;            // rows of a CTA, of equal number
    gy = (B + each - 1) / each;
  }
  *rows = (int)gy;
  (void)dtype;
}

cudaError_t launch_gated_fwd(const GatedParams& p, cudaStream_t s) {
  return p.dtype == M3_BF16 ? fwd_impl<__nv_bfloat16>(p, s) : fwd_impl<float>(p, s);
}

cudaError_t launch_gated_step(const GatedStepParams& p, cudaStream_t s) {
  const int e = dsize(p.dtype);
  const bool v4 = p.D % 4 == 0 && p.ld_x % 4 == 0 && p.ld_r % 4 == 0 && p.ld_i % 4 == 0 &&
                  aligned(p.h, 16) && aligned(p.x, 4 * e) && aligned(p.rg, 4 * e) &&
                  aligned(p.ig, 4 * e) && aligned(p.y, 4 * e);
  if (p.dtype == M3_BF16)
    return v4 ? step_impl<__nv_bfloat16, 4>(p, s) : step_impl<__nv_bfloat16, 1>(p, s);
  return v4 ? step_impl<float, 4>(p, s) : step_impl<float, 1>(p, s);
}

}  // namespace m3
