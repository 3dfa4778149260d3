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

#ifndef M3_GF
#define M3_GF 3
#endif
#ifndef M3_GS
#define M3_GS 8
#endif
#ifndef M3_GL
#define M3_GL 8
#endif
namespace m3 {
namespace {

__device__ __forceinline__ int row_length(const int* lengths, int b, int L) {
  if (lengths == nullptr) return L;
  const int n = lengths[b];
  return n < 0 ? 0 : n > L ? L : n;
}

template <typename T, int LC, int TS>
__global__ void __launch_bounds__(32 * kGatedWarps, M3_GF) gated_fwd_kernel(const GatedParams p) {
  extern __shared__ __align__(16) char smem[];
  __shared__ Joint<LC> joint;
  using St = Stage<T, 3, LC, TS>;
  using La = Lanes<LC, TS>;
  const int lane = threadIdx.x, w = __shfl_sync(0xffffffffu, threadIdx.y, 0), W = blockDim.y;
  const int S = p.splits, rank = blockIdx.x % S;
  const int c0 = blockIdx.x / S * La::kTile, c = c0 + lane % LC * 2;
  const int left = p.D - c, D = p.D, L = p.L, span = S * W * La::kSteps;
  const int tw0 = (rank * W + w) * La::kSteps, own = lane / LC * TS;   // of the warp; of the run
  const bool vec = p.vec != 0;
  const long long ld[3] = {p.ld_x, p.ld_r, p.ld_i};
  char* buf = smem + w * St::kBytes;
  St st;
  const float2 dec = load_pair(p.decay + c, left);
  const float2 k = make_float2(-p.c * softplus_f(dec.x), -p.c * softplus_f(dec.y));
  const bool near = __all_sync(0xffffffffu, k.x >= -kNear && k.y >= -kNear);
  int flip = 0;
  if (S > 1) cluster_sync();                         // every CTA runs before its memory is written
  // the copies of a row's first pass start while the row before it is finished
  auto start = [&](int b, int n) {
    const long long row = (long long)b * L + tw0;
    st.at(0, p.x, row, ld[0], c0, vec);
    st.at(1, p.rg, row, ld[1], c0, vec);
    st.at(2, p.ig, row, ld[2], c0, vec);
    st.issue(buf, ld, tw0, n, c0, D, vec);
  };
  int n = row_length(p.lengths, blockIdx.y, L), n2;
  if (n > 0) start(blockIdx.y, n);
  for (int b = blockIdx.y; b < p.B; b += gridDim.y, n = n2) {
    const int nb = b + gridDim.y;
    n2 = nb < p.B ? row_length(p.lengths, nb, L) : 0;
    float2 carry = p.h0 != nullptr ? load_pair(p.h0 + (size_t)b * D + c, left) : f2(0.f);
    if (n == 0) {
      if (n2 > 0) start(nb, n2);
      if (p.h_last != nullptr && rank == 0 && w == 0 && lane < LC)
        store_pair(p.h_last + (size_t)b * D + c, carry, left, false);
    }
    int tw = tw0;
    T* y = static_cast<T*>(p.y) + ((size_t)b * L + tw0 + own) * D + c;
    float* ck = p.ckpt == nullptr ? nullptr
                                  : p.ckpt + ((size_t)b * ((L + kGatedCkpt - 1) / kGatedCkpt) +
                                              (tw0 + own) / kGatedCkpt) * D + c;
    for (int s0 = 0; s0 < n; s0 += span, tw += span) {
      const int t0 = tw + own;
      St::wait();
      // FAST: every step of the warp is one of the sequence, and no decay is far from 1
      auto pass = [&](auto fast) {
        constexpr bool FAST = decltype(fast)::value;
        float2 a[TS], v[TS];
        Run run{f2(1.f), f2(0.f)};
#pragma unroll
        for (int i = 0; i < TS; ++i) {
          const float2 x = St::get(buf, 0, i), r = sigmoid2(St::get(buf, 1, i)),
                       g = sigmoid2(St::get(buf, 2, i));
          float2 m, inv;
          decay2<FAST>(mul2(k, r), a[i], m);
          root2(m, m, inv);
          v[i] = mul2(mul2(m, g), x);
          if (!FAST && t0 + i >= n) {                // the state stays
            a[i] = f2(1.f);
            v[i] = f2(0.f);
          }
          run.V = fma2(a[i], run.V, v[i]);
          run.P = mul2(a[i], run.P);
        }
        __syncwarp();
        if (s0 + span < n) {
#pragma unroll
          for (int q = 0; q < 3; ++q) st.p[q] += (long long)span * ld[q];
          st.issue(buf, ld, tw + span, n, c0, D, vec);
        } else if (n2 > 0) {
          start(nb, n2);
        }
        float2 h = join<LC, 1>(joint, flip, run, w, W, rank, S, s0 == 0, carry);
#pragma unroll
        for (int i = 0; i < TS; ++i) {
          if (i % kGatedCkpt == 0 && ck != nullptr && (FAST || t0 + i < n))
            store_pair(ck + (size_t)(i / kGatedCkpt) * D, h, left, D % 2 == 0);
          h = fma2(a[i], h, v[i]);
          if (FAST) store_pair(y + (size_t)i * D, h, left, vec);
          else if (t0 + i < L) store_pair(y + (size_t)i * D, t0 + i < n ? h : f2(0.f), left, vec);
        }
      };
      if (near && tw + La::kSteps <= n) pass(std::true_type());
      else pass(std::false_type());
      flip ^= 1;
      y += (size_t)span * D;
      if (ck != nullptr) ck += (size_t)(span / kGatedCkpt) * D;
    }
    if (n > 0 && p.h_last != nullptr && rank == 0 && w == W - 1 && lane >= 32 - LC)
      store_pair(p.h_last + (size_t)b * D + c, carry, left, false);
    for (; tw - tw0 < L; tw += span) {               // steps past the length
      for (int i = 0; i < TS && tw + own + i < L; ++i)
        store_pair(y + (size_t)i * D, f2(0.f), left, vec);
      y += (size_t)span * D;
    }
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
      decay2<false>(mul2(make_float2(k[j], k[j + o]),
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

template <typename T, int LC>
cudaError_t fwd_impl(const GatedParams& p, cudaStream_t s) {
  constexpr int TS = kGatedFwdSteps, kBytes = Stage<T, 3, LC, TS>::kBytes, kTile = 2 * LC;
  const cudaError_t e = allow_smem<gated_fwd_kernel<T, LC, TS>>(kGatedWarps * kBytes);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((p.D + kTile - 1) / kTile * p.splits), p.rows);
  cfg.blockDim = dim3(32, p.warps);
  cfg.dynamicSmemBytes = p.warps * kBytes;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = p.splits > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, gated_fwd_kernel<T, LC, TS>, p);
}

template <typename T>
cudaError_t fwd_lanes(const GatedParams& p, cudaStream_t s) {
  if (p.lanes == 32) return fwd_impl<T, 32>(p, s);
  return p.lanes == 16 ? fwd_impl<T, 16>(p, s) : fwd_impl<T, 8>(p, s);
}

}  // namespace

int gated_segments(int L) { return (L + kGatedCkpt - 1) / kGatedCkpt; }

void gated_plan(int B, int L, int D, bool backward, int sms, GatedParams* p) {
  const int per = backward ? M3_GB : M3_GF;                 // CTAs per SM
  const int ts = backward ? kGatedBwdSteps : kGatedFwdSteps, segs = (L + ts - 1) / ts;
  const long long wave = (long long)per * sms;
  const int warps = segs < kGatedWarps ? segs : kGatedWarps;
  // Of the tile widths and time splits whose every CTA has a pass of its own, the one
  // with most CTAs in one wave; wide tiles and few splits among equals.
  int lanes = 32, S = 1;
  auto tiles = [&](int l) { return (long long)(D + 2 * l - 1) / (2 * l); };
  long long most = tiles(32) * B;
  for (int l = 32; l >= M3_GL; l /= 2)
    for (int k = 1; k <= M3_GS; ++k) {
      const long long ctas = tiles(l) * B * k;
      if (ctas <= wave && ctas > most && segs >= (long long)k * warps * (32 / l)) {
        most = ctas;
        lanes = l;
        S = k;
      }
    }
  p->lanes = lanes;
  p->warps = warps;
  p->splits = S;
  long long gy = B, cap = wave / (tiles(lanes) * S);
  if (cap < 1) cap = 1;
  if (cap > 65535) cap = 65535;
  if (gy > cap) {
    const long long each = (B + cap - 1) / cap;            // rows of a CTA, of equal number
    gy = (B + each - 1) / each;
  }
  p->rows = (int)gy;
}

cudaError_t launch_gated_fwd(const GatedParams& p, cudaStream_t s) {
  return p.dtype == M3_BF16 ? fwd_lanes<__nv_bfloat16>(p, s) : fwd_lanes<float>(p, s);
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
