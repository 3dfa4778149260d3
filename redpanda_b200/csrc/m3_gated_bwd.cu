// Gated linear recurrence, backward.  Formulas of the forward: m3_gated.cuh.
//
//   q_t   = g_t + a_{t+1} q_{t+1}                        (gradient of h_t)
//   dx_t  = q m i,   dig_t = q m x i (1 - i)
//   e_t   = q l (a h_{t-1} - (a^2 / m) i x)              (l times the gradient of l)
//   drg_t = e (1 - r),   ddecay = sigmoid(decay) / softplus(decay) sum e
// l / m is finite where l goes to 0 (a gate far closed), the gradient of l itself
// is not, so only the product is formed.
//
// As in the forward's second kernel a thread holds a run of steps, here 4, the warps
// and the cluster's CTAs consecutive runs, and the passes go from the sequence's end to
// its start.  The forward's checkpoint in front of every run gives h_{t-1} in fp32 (y
// in bf16 would put its rounding on e); a thread computes forward what multiplies q in
// each gradient, then joins the runs behind its own and walks back with q.  ddecay
// stays in registers over all steps of a thread; each CTA writes one partial per
// channel, and a second launch adds them in a fixed order.
//
// Seven arrays and the checkpoints (1 byte per element) move: 256 x 64 x 2048 bf16 105
// us (4.8 TB/s), at half of the issue slots with 16 warps per SM of 128 registers (96
// registers for more warps spill: 121 us; a warp per row without joins spills at 96 and
// is slower at 128: 123 us).  2 x 16001 x 1280 fp32: 200 us (5.7 TB/s).
#include "m3_gated.cuh"

#include <type_traits>

#include "m3_api_util.h"
#include "m3_common.cuh"
#include "m3_ops.h"
#include "m3_pdl.cuh"

namespace m3 {
namespace {

__device__ __forceinline__ int row_length(const int* lengths, int b, int L) {
  if (lengths == nullptr) return L;
  const int n = lengths[b];
  return n < 0 ? 0 : n > L ? L : n;
}

// What multiplies q in the gradients of a step, and the step of h
struct Factors {
  float2 a, X, I, A, R;
};
template <bool FAST>
__device__ __forceinline__ Factors factors(float2 k, float2 x, float2 rg, float2 ig, float2& h) {
  const float2 r = sigmoid2(rg), u = sigmoid2(ig), l = mul2(k, r);
  float2 m, inv;
  Factors f;
  decay2<FAST>(l, f.a, m);
  root2(m, m, inv);
  const float2 ah = mul2(f.a, h), ux = mul2(u, x), am = mul2(mul2(f.a, f.a), inv);
  f.X = mul2(m, u);
  h = fma2(m, ux, ah);
  f.A = mul2(l, fma2(mul2(am, f2(-1.f)), ux, ah));
  f.R = fma2(r, f2(-1.f), f2(1.f));
  f.I = mul2(mul2(f.X, x), fma2(u, f2(-1.f), f2(1.f)));
  return f;
}

template <typename T, int LC, int TS, int MODE>
__global__ void __launch_bounds__(256, 2)
    gated_bwd_kernel(const GatedBwdParams q) {
  extern __shared__ __align__(16) char smem[];
  static_assert(TS == kGatedCkpt, "a run starts at a checkpoint");
  using St = Stage<T, 4, LC, TS, MODE>;
  using La = Lanes<LC, TS>;
  const GatedParams& p = q.f;
  const int lane = threadIdx.x, w = __shfl_sync(0xffffffffu, threadIdx.y, 0), W = blockDim.y;
  const int S = p.splits, rank = blockIdx.x % S;
  const int c0 = blockIdx.x / S * La::kTile, c = c0 + St::channel();
  const int left = p.D - c, D = p.D, L = p.L, span = S * W * La::kSteps;
  const int tw0 = (rank * W + w) * La::kSteps, own = lane / LC * TS;   // of the warp; of the run
  const long long ld[4] = {p.ld_x, p.ld_r, p.ld_i, D};
  const long long rows = (long long)p.B * L;
  const void* const bases[4] = {p.x, p.rg, p.ig, q.g};
  char* buf = smem + w * St::kBytes;
  const Joint<LC> joint(smem + W * St::kBytes, W, S);
  St st;
  const float2 k = rates<St>(p.decay + c, p.c, left);
  const bool near = __all_sync(0xffffffffu, k.x >= -kNear && k.y >= -kNear);
  float2 sum = f2(0.f);
  int turn = 0;
  bool dead = false;
  joint.start();
  // the copies of a row's first pass, its last steps, start while the row before it
  // is finished
  auto start = [&](int b, int n) {
    const int tw = (n - 1) / span * span + tw0;
    const long long row = (long long)b * L + tw;
    st.at(0, p.x, row, ld[0], c0);
    st.at(1, p.rg, row, ld[1], c0);
    st.at(2, p.ig, row, ld[2], c0);
    st.at(3, q.g, row, ld[3], c0);
    st.issue(buf, bases, ld, rows, tw, n, c0, D);
  };
  int n = row_length(p.lengths, blockIdx.y, L), n2;
  if (n > 0) start(blockIdx.y, n);
  for (int b = blockIdx.y; b < p.B; b += gridDim.y, n = n2) {
    const int nb = b + gridDim.y;
    n2 = nb < p.B ? row_length(p.lengths, nb, L) : 0;
    if (n == 0 && n2 > 0) start(nb, n2);
    const long long base = (long long)b * L;
    const int passes = (n + span - 1) / span;
    // steps of passes that are wholly past the length
    for (int t0 = passes * span + tw0 + own; t0 - tw0 - own < L; t0 += span)
      for (int i = 0; i < TS && t0 + i < L; ++i) {
        const size_t at = (size_t)(base + t0 + i) * D + c;
        store_pair<St>(static_cast<T*>(q.dx) + at, f2(0.f), left);
        store_pair<St>(static_cast<T*>(q.drg) + at, f2(0.f), left);
        store_pair<St>(static_cast<T*>(q.dig) + at, f2(0.f), left);
      }
    float2 carry = f2(0.f);                          // a_{t+1} q_{t+1}
    int tw = (passes - 1) * span + tw0;
    size_t at = (size_t)(base + tw + own) * D + c;
    const float* ck = p.ckpt + ((size_t)b * ((L + TS - 1) / TS) + (tw + own) / TS) * D + c;
    // (a row without steps has no pass, and tw lies before it)
    float2 h = passes > 0 && tw + own < n ? load_each<St>(ck, left) : f2(0.f);
    for (int k0 = passes; k0 > 0; --k0, tw -= span) {
      const int t0 = tw + own;
      const auto shift = St::shifts(bases, ld, base + t0, c0);
      St::wait();
      // FAST: every step of the warp is one of the sequence, and no decay is far from 1
      auto pass = [&](auto fast) {
        constexpr bool FAST = decltype(fast)::value;
        float2 a[TS], X[TS], I[TS], A[TS], R[TS], g[TS];
#pragma unroll
        for (int i = 0; i < TS; ++i) {
          const Factors f = factors<FAST>(k, St::get(buf, 0, i, shift), St::get(buf, 1, i, shift),
                                          St::get(buf, 2, i, shift), h);
          g[i] = St::get(buf, 3, i, shift);
          a[i] = f.a, X[i] = f.X, I[i] = f.I, A[i] = f.A, R[i] = f.R;
          if (!FAST && t0 + i >= n) {                // the state stays, nothing has a gradient
            a[i] = f2(1.f);
            g[i] = X[i] = I[i] = A[i] = R[i] = f2(0.f);
          }
        }
        Run run{f2(1.f), f2(0.f)};                   // v = a (g + v), from the last step
#pragma unroll
        for (int i = TS - 1; i >= 0; --i) {
          run.V = mul2(a[i], add2(g[i], run.V));
          run.P = mul2(a[i], run.P);
        }
        __syncwarp();
        if (k0 > 1) {
#pragma unroll
          for (int z = 0; z < 4; ++z) st.p[z] -= (long long)span * ld[z];
          st.issue(buf, bases, ld, rows, tw - span, n, c0, D);
          ck -= (size_t)(span / TS) * D;
          h = load_each<St>(ck, left);                   // every pass but the last is full
        } else if (n2 > 0) {
          start(nb, n2);
        }
        float2 v = join<LC, -1>(joint, turn, run, W - 1 - w, S - 1 - rank, k0 == passes, carry,
                                    dead);
        float2 part = f2(0.f);
#pragma unroll
        for (int i = TS - 1; i >= 0; --i) {
          const float2 qt = add2(g[i], v), e = mul2(qt, A[i]);
          v = mul2(a[i], qt);
          part = add2(part, e);
          if (FAST || t0 + i < L) {
            const size_t o = at + (size_t)i * D;
            store_pair<St>(static_cast<T*>(q.dx) + o, mul2(qt, X[i]), left);
            store_pair<St>(static_cast<T*>(q.drg) + o, mul2(e, R[i]), left);
            store_pair<St>(static_cast<T*>(q.dig) + o, mul2(qt, I[i]), left);
          }
        }
        sum = add2(sum, part);
      };
      if (near && tw + La::kSteps <= n) pass(std::true_type());
      else pass(std::false_type());
      ++turn;
      at -= (size_t)span * D;
    }
  }
  if (S > 1) cluster_sync();                         // nobody writes to a CTA that has left
  if (dead) set_err(p.err, M3_ERR_DEVICE);
  pdl_launch_dependents();
  // the CTA's partial: the runs of a warp, then the warps, in order
#pragma unroll
  for (int s = LC; s < 32; s *= 2)
    sum = add2(sum, make_float2(__shfl_xor_sync(0xffffffffu, sum.x, s),
                                __shfl_xor_sync(0xffffffffu, sum.y, s)));
  __syncthreads();
  float2* s = reinterpret_cast<float2*>(smem);
  if (lane < LC) s[w * LC + lane] = sum;
  __syncthreads();
  if (w == 0 && lane < LC) {
    float2 v = s[lane];
    for (int i = 1; i < W; ++i) v = add2(v, s[i * LC + lane]);
    store_each<St>(q.part + ((size_t)blockIdx.y * S + rank) * D + c, v, left);
  }
}

// ddecay[c] = sigmoid(decay) / softplus(decay) * the sum of the CTAs' partials: 32
// columns per CTA, 32 strided sums each, joined in order.
__global__ void __launch_bounds__(1024) gated_reduce_kernel(const float* part, int n, int D,
                                                            const float* decay, float* out) {
  __shared__ float s[32][33];
  const int cx = threadIdx.x & 31, k = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + cx;
  float a = 0.f;
  pdl_wait();
  if (c < D)
    for (int i = k; i < n; i += 32) a += part[(size_t)i * D + c];
  s[k][cx] = a;
  __syncthreads();
  float v = s[cx][k];
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  const int cc = blockIdx.x * 32 + k;
  if (cx == 0 && cc < D) {
    const float d = decay[cc], e = expf(-fabsf(d));
    // both go as e^d far below 0, where their ratio is 1
    out[cc] = d < -15.f ? v : v * ((d < 0.f ? e : 1.f) / (1.f + e)) / softplus_f(d);
  }
}

cudaError_t reduce(const GatedBwdParams& q, cudaStream_t s) {
  const GatedParams& p = q.f;
  return launch_maybe_pdl(true, gated_reduce_kernel, dim3((p.D + 31) / 32), dim3(1024), 0, s,
                          (const float*)q.part, p.rows * p.splits, p.D, p.decay, q.ddecay);
}

template <typename T, int LC, int MODE>
cudaError_t bwd_impl(const GatedBwdParams& q, cudaStream_t s) {
  constexpr int TS = kGatedBwdSteps, kBytes = Stage<T, 4, LC, TS, MODE>::kBytes, kTile = 2 * LC;
  const GatedParams& p = q.f;
  const cudaError_t e = allow_smem<gated_bwd_kernel<T, LC, TS, MODE>>(
      kGatedWarps * kBytes + joint_bytes(LC, kGatedWarps, 8));
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((p.D + kTile - 1) / kTile * p.splits), p.rows);
  cfg.blockDim = dim3(32, p.warps);
  cfg.dynamicSmemBytes = p.warps * kBytes + joint_bytes(LC, p.warps, p.splits);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = p.splits > 1 ? 1 : 0;
  const cudaError_t r = cudaLaunchKernelEx(&cfg, gated_bwd_kernel<T, LC, TS, MODE>, q);
  return r != cudaSuccess ? r : reduce(q, s);
}

template <typename T, int MODE>
cudaError_t bwd_lanes(const GatedBwdParams& q, cudaStream_t s) {
  if (q.f.lanes == 32) return bwd_impl<T, 32, MODE>(q, s);
  return q.f.lanes == 16 ? bwd_impl<T, 16, MODE>(q, s) : bwd_impl<T, 8, MODE>(q, s);
}

}  // namespace

int gated_bwd_in_clusters(int k) {
  static OncePerDevice known[9];
  constexpr int kBytes = Stage<float, 4, 32, kGatedBwdSteps, kVectors>::kBytes;
  return resident_in_clusters<gated_bwd_kernel<float, 32, kGatedBwdSteps, kVectors>>(
      known[k], k, kGatedWarps * kBytes + joint_bytes(32, kGatedWarps, k));
}

cudaError_t launch_gated_bwd(const GatedBwdParams& q, cudaStream_t s) {
  const int copy = q.f.copy;
  if (q.f.dtype == M3_F32)
    return copy == kVectors ? bwd_lanes<float, kVectors>(q, s) : bwd_lanes<float, kWords>(q, s);
  using B = __nv_bfloat16;
  return copy == kVectors ? bwd_lanes<B, kVectors>(q, s)
         : copy == kWords ? bwd_lanes<B, kWords>(q, s)
                          : bwd_lanes<B, kAny>(q, s);
}

}  // namespace m3
