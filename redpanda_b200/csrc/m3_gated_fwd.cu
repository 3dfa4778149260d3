// Gated linear recurrence, forward over whole sequences and single tokens.
// Formulas and the precision of the decay: m3_gated.cuh.
//
// Bound by memory (x and the gates in, y out) and by the MUFU unit (two exponentials,
// two reciprocals and a root per element: 37 us at 256 x 64 x 2048, 41 us of bf16
// bytes).  Two kernels:
//
// Where rows and channel tiles give every warp of the GPU its own, a warp walks 64
// channels of a row by itself, 4 steps at a time, the next ones' copies in flight;
// nothing is stored but y.  256 x 64 x 2048 bf16: 56 us (4.8 TB/s; MUFU 73 % busy), 65
// us with two warps per row that are joined.
//
// With fewer, a CTA holds a tile of 64, 32 or 16 channels, two per lane, and its warps
// hold consecutive runs of 8 steps; a cluster of up to 8 CTAs holds that many runs
// more.  Each pass of a CTA (cluster) over its runs loads every input once: a thread
// computes a and b = m i x of its steps, the run's product and sum, joins the runs
// ahead (join()), and walks its steps from there; the copies of the next pass's rows
// are in flight meanwhile.  One prompt of 16384 x 1024 bf16: 50 us (2.7 TB/s), 11
// passes of 4.5 us each, of which half is the wait for the runs ahead and for the
// slowest warp; 101 us with tiles of 64 channels only (before
// mbarriers).
#include "m3_gated.cuh"

#include <type_traits>

#include "m3_api_util.h"
#include "m3_common.cuh"
#include "m3_ops.h"

namespace m3 {
namespace {

__device__ __forceinline__ int row_length(const int* lengths, int b, int L) {
  if (lengths == nullptr) return L;
  const int n = lengths[b];
  return n < 0 ? 0 : n > L ? L : n;
}

template <typename T, int LC, int TS, int MODE>
__global__ void __launch_bounds__(256, 3) gated_fwd_kernel(const GatedParams p) {
  extern __shared__ __align__(16) char smem[];
  using St = Stage<T, 3, LC, TS, MODE>;
  using La = Lanes<LC, TS>;
  const int lane = threadIdx.x, w = __shfl_sync(0xffffffffu, threadIdx.y, 0), W = blockDim.y;
  const int S = p.splits, rank = blockIdx.x % S;
  const int c0 = blockIdx.x / S * La::kTile, c = c0 + St::channel();
  const int left = p.D - c, D = p.D, L = p.L, span = S * W * La::kSteps;
  const int tw0 = (rank * W + w) * La::kSteps, own = lane / LC * TS;   // of the warp; of the run
  const long long ld[3] = {p.ld_x, p.ld_r, p.ld_i};
  const long long rows = (long long)p.B * L;
  const void* const base[3] = {p.x, p.rg, p.ig};
  char* buf = smem + w * St::kBytes;
  const Joint<LC> joint(smem + W * St::kBytes, W, S);
  St st;
  const float2 k = rates<St>(p.decay + c, p.c, left);
  const bool near = __all_sync(0xffffffffu, k.x >= -kNear && k.y >= -kNear);
  int turn = 0;
  bool dead = false;
  joint.start();
  // the copies of a row's first pass start while the row before it is finished
  auto start = [&](int b, int n) {
    const long long row = (long long)b * L + tw0;
    st.at(0, p.x, row, ld[0], c0);
    st.at(1, p.rg, row, ld[1], c0);
    st.at(2, p.ig, row, ld[2], c0);
    st.issue(buf, base, ld, rows, tw0, n, c0, D);
  };
  int n = row_length(p.lengths, blockIdx.y, L), n2;
  if (n > 0) start(blockIdx.y, n);
  for (int b = blockIdx.y; b < p.B; b += gridDim.y, n = n2) {
    const int nb = b + gridDim.y;
    n2 = nb < p.B ? row_length(p.lengths, nb, L) : 0;
    float2 carry = p.h0 != nullptr ? load_each<St>(p.h0 + (size_t)b * D + c, left) : f2(0.f);
    if (n == 0) {
      if (n2 > 0) start(nb, n2);
      if (p.h_last != nullptr && rank == 0 && w == 0 && lane < LC)
        store_each<St>(p.h_last + (size_t)b * D + c, carry, left);
    }
    int tw = tw0;
    T* y = static_cast<T*>(p.y) + ((size_t)b * L + tw0 + own) * D + c;
    float* ck = p.ckpt == nullptr ? nullptr
                                  : p.ckpt + ((size_t)b * ((L + kGatedCkpt - 1) / kGatedCkpt) +
                                              (tw0 + own) / kGatedCkpt) * D + c;
    for (int s0 = 0; s0 < n; s0 += span, tw += span) {
      const int t0 = tw + own;
      const auto shift = St::shifts(base, ld, (long long)b * L + t0, c0);
      St::wait();
      // FAST: every step of the warp is one of the sequence, and no decay is far from 1
      auto pass = [&](auto fast) {
        constexpr bool FAST = decltype(fast)::value;
        float2 a[TS], v[TS];
        Run run{f2(1.f), f2(0.f)};
#pragma unroll
        for (int i = 0; i < TS; ++i) {
          const float2 x = St::get(buf, 0, i, shift), r = sigmoid2(St::get(buf, 1, i, shift)),
                       g = sigmoid2(St::get(buf, 2, i, shift));
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
          st.issue(buf, base, ld, rows, tw + span, n, c0, D);
        } else if (n2 > 0) {
          start(nb, n2);
        }
        float2 h = join<LC, 1>(joint, turn, run, w, rank, s0 == 0, carry, dead);
#pragma unroll
        for (int i = 0; i < TS; ++i) {
          if (i % kGatedCkpt == 0 && ck != nullptr && (FAST || t0 + i < n))
            store_pair<St>(ck + (size_t)(i / kGatedCkpt) * D, h, left);
          h = fma2(a[i], h, v[i]);
          if (FAST) store_pair<St>(y + (size_t)i * D, h, left);
          else if (t0 + i < L) store_pair<St>(y + (size_t)i * D, t0 + i < n ? h : f2(0.f), left);
        }
      };
      if (near && tw + La::kSteps <= n) pass(std::true_type());
      else pass(std::false_type());
      ++turn;
      y += (size_t)span * D;
      if (ck != nullptr) ck += (size_t)(span / kGatedCkpt) * D;
    }
    if (n > 0 && p.h_last != nullptr && rank == 0 && w == W - 1 && lane >= 32 - LC)
      store_each<St>(p.h_last + (size_t)b * D + c, carry, left);
    for (; tw - tw0 < L; tw += span) {               // steps past the length
      for (int i = 0; i < TS && tw + own + i < L; ++i)
        store_pair<St>(y + (size_t)i * D, f2(0.f), left);
      y += (size_t)span * D;
    }
  }
  if (S > 1) cluster_sync();                         // nobody writes to a CTA that has left
  if (dead) set_err(p.err, M3_ERR_DEVICE);
}

// Many rows: a warp walks 64 channels of a row by itself, so that there is nothing
// to join; the CTA's warps are workers of their own.  Two buffers of 4 steps.
template <typename T, int MODE>
__global__ void __launch_bounds__(128, 8) gated_rows_fwd_kernel(const GatedParams p) {
  extern __shared__ __align__(16) char smem[];
  constexpr int TS = 4;
  static_assert(TS == kGatedCkpt, "a pass starts at a checkpoint");
  using St = Stage<T, 3, 32, TS, MODE>;
  const int w = threadIdx.y;
  const int c0 = blockIdx.x * 64, c = c0 + St::channel(), left = p.D - c, D = p.D, L = p.L;
  const long long ld[3] = {p.ld_x, p.ld_r, p.ld_i};
  const long long rows = (long long)p.B * L;
  const void* const base[3] = {p.x, p.rg, p.ig};
  char* buf = smem + w * 2 * St::kBytes;
  St st;
  const int step = gridDim.y * blockDim.y;
  int b = blockIdx.y * blockDim.y + w, nb, n, tn = 0;   // (nb, tn): the pass that is copied next
  if (b >= p.B) return;
  auto at = [&](int row) {
    st.at(0, p.x, (long long)row * L, ld[0], c0);
    st.at(1, p.rg, (long long)row * L, ld[1], c0);
    st.at(2, p.ig, (long long)row * L, ld[2], c0);
  };
  nb = b;
  int nn = n = row_length(p.lengths, b, L);             // the length of nb
  at(b);
  int put = 0, get = 0;
  // copies the next pass, of this row or of the next that has one
  auto ahead = [&] {
    while (tn >= nn && nb < p.B) {
      nb += step;
      tn = 0;
      if (nb < p.B) {
        nn = row_length(p.lengths, nb, L);
        at(nb);
      }
    }
    if (nb < p.B) {
      st.issue(buf + put * St::kBytes, base, ld, rows, tn, nn, c0, D);
#pragma unroll
      for (int q = 0; q < 3; ++q) st.p[q] += TS * ld[q];
      tn += TS;
      put ^= 1;
    } else {
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  };
  ahead();
  const float2 k = rates<St>(p.decay + c, p.c, left);
  const bool near = __all_sync(0xffffffffu, k.x >= -kNear && k.y >= -kNear);
  for (; b < p.B; b += step) {
    n = row_length(p.lengths, b, L);
    float2 h = p.h0 != nullptr ? load_each<St>(p.h0 + (size_t)b * D + c, left) : f2(0.f);
    T* y = static_cast<T*>(p.y) + (size_t)b * L * D + c;
    float* ck = p.ckpt == nullptr ? nullptr : p.ckpt + (size_t)b * ((L + TS - 1) / TS) * D + c;
    for (int t0 = 0; t0 < n; t0 += TS) {
      ahead();
      const auto shift = St::shifts(base, ld, (long long)b * L + t0, c0);
      St::template wait<1>();
      const char* from = buf + get * St::kBytes;
      get ^= 1;
      if (ck != nullptr) {
        store_pair<St>(ck, h, left);
        ck += D;
      }
      auto pass = [&](auto fast) {
        constexpr bool FAST = decltype(fast)::value;
#pragma unroll
        for (int i = 0; i < TS; ++i) {
          const float2 x = St::get(from, 0, i, shift), r = sigmoid2(St::get(from, 1, i, shift)),
                       g = sigmoid2(St::get(from, 2, i, shift));
          float2 a, m, inv;
          decay2<FAST>(mul2(k, r), a, m);
          root2(m, m, inv);
          const float2 v = fma2(a, h, mul2(mul2(m, g), x));
          if (FAST || t0 + i < n) {
            h = v;
            store_pair<St>(y, h, left);
            y += D;
          }
        }
      };
      if (near && t0 + TS <= n) pass(std::true_type());
      else pass(std::false_type());
      __syncwarp();
    }
    if (p.h_last != nullptr) store_each<St>(p.h_last + (size_t)b * D + c, h, left);
    for (int t = n; t < L; ++t, y += D) store_pair<St>(y, f2(0.f), left);
  }
}

// One token per row: a thread owns V channels and walks rows, the next row's loads
// ahead of the present one's arithmetic.  Bound by memory: 2048 x 2048 bf16 14 us (4.8
// TB/s), fp32 19 us (5.2 TB/s).  Rows that vectors of 4 do not fit go by elements, bound
// by the number of accesses: 2048 x 2046 and x 2047 bf16 20 us, x 2047 fp32 26 us.
template <typename T, int V>
struct StepRow {
  Pack<T, V> x, r, g;
  Pack<float, V> h;
  __device__ __forceinline__ void load(const GatedStepParams& p, int b, int c) {
    x = ld_pack<T, V>(static_cast<const T*>(p.x) + (size_t)b * p.ld_x + c);
    r = ld_pack<T, V>(static_cast<const T*>(p.rg) + (size_t)b * p.ld_r + c);
    g = ld_pack<T, V>(static_cast<const T*>(p.ig) + (size_t)b * p.ld_i + c);
    h = ld_pack<float, V>(p.h + (size_t)b * p.D + c);
  }
};
template <typename T, int V>
__global__ void __launch_bounds__(256) gated_step_kernel(const GatedStepParams p) {
  const int c = (blockIdx.x * 32 + threadIdx.x) * V;
  int b = blockIdx.y * blockDim.y + threadIdx.y;
  const int step = gridDim.y * blockDim.y;
  if (c >= p.D || b >= p.B) return;
  StepRow<T, V> now;
  now.load(p, b, c);
  float k[V];
#pragma unroll
  for (int j = 0; j < V; ++j) k[j] = -p.c * softplus_f(p.decay[c + j]);
  for (; b < p.B; b += step) {
    StepRow<T, V> next;
    if (b + step < p.B) next.load(p, b + step, c);
    Pack<float, V> h;
    Pack<T, V> y;
    y.zero();
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      constexpr int o = V > 1 ? 1 : 0;
      float2 a, m, inv;
      decay2<false>(mul2(make_float2(k[j], k[j + o]),
                         sigmoid2(make_float2(now.r.get(j), now.r.get(j + o)))), a, m);
      root2(m, m, inv);
      const float2 in = mul2(mul2(m, sigmoid2(make_float2(now.g.get(j), now.g.get(j + o)))),
                             make_float2(now.x.get(j), now.x.get(j + o)));
      const float2 q = fma2(a, make_float2(now.h.get(j), now.h.get(j + o)), in);
      h.put(j, q.x);
      y.put(j, q.x);
      if (V > 1) {
        h.put(j + o, q.y);
        y.put(j + o, q.y);
      }
    }
    st_pack<float, V>(p.h + (size_t)b * p.D + c, h);
    st_pack<T, V>(static_cast<T*>(p.y) + (size_t)b * p.D + c, y);
    now = next;
  }
}

template <typename T, int V>
cudaError_t step_impl(const GatedStepParams& p, cudaStream_t s) {
  static OncePerDevice known;
  const int tiles = (p.D + 32 * V - 1) / (32 * V);
  const int ty = p.B < 8 ? p.B : 8;
  // one wave of CTAs, of rows in equal number
  const int per = resident_ctas<gated_step_kernel<T, V>>(known, 256, 0);
  if (per <= 0) return cudaErrorInvalidConfiguration;
  long long gy = (p.B + ty - 1) / ty, cap = (long long)per * p.sms / tiles;
  cap = cap < 1 ? 1 : cap > 65535 ? 65535 : cap;
  if (gy > cap) {
    const long long each = (gy + cap - 1) / cap;
    gy = (gy + each - 1) / each;
  }
  gated_step_kernel<T, V><<<dim3(tiles, (unsigned)gy), dim3(32, ty), 0, s>>>(p);
  return cudaGetLastError();
}

template <typename T, int LC, int MODE>
cudaError_t fwd_impl(const GatedParams& p, cudaStream_t s) {
  constexpr int TS = kGatedFwdSteps, kBytes = Stage<T, 3, LC, TS, MODE>::kBytes, kTile = 2 * LC;
  const cudaError_t e = allow_smem<gated_fwd_kernel<T, LC, TS, MODE>>(
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
  return cudaLaunchKernelEx(&cfg, gated_fwd_kernel<T, LC, TS, MODE>, p);
}

template <typename T, int MODE>
cudaError_t fwd_rows(const GatedParams& p, cudaStream_t s) {
  constexpr int kBytes = 2 * Stage<T, 3, 32, 4, MODE>::kBytes;
  const cudaError_t e = allow_smem<gated_rows_fwd_kernel<T, MODE>>(4 * kBytes);
  if (e != cudaSuccess) return e;
  gated_rows_fwd_kernel<T, MODE>
      <<<dim3((p.D + 63) / 64, p.rows), dim3(32, p.warps), p.warps * kBytes, s>>>(p);
  return cudaGetLastError();
}

template <typename T, int MODE>
cudaError_t fwd_lanes(const GatedParams& p, cudaStream_t s) {
  if (p.solo) return fwd_rows<T, MODE>(p, s);
  if (p.lanes == 32) return fwd_impl<T, 32, MODE>(p, s);
  return p.lanes == 16 ? fwd_impl<T, 16, MODE>(p, s) : fwd_impl<T, 8, MODE>(p, s);
}

}  // namespace

static int fwd_in_clusters(int k) {
  static OncePerDevice known[9];
  constexpr int kBytes = Stage<float, 3, 32, kGatedFwdSteps, kVectors>::kBytes;
  return resident_in_clusters<gated_fwd_kernel<float, 32, kGatedFwdSteps, kVectors>>(
      known[k], k, kGatedWarps * kBytes + joint_bytes(32, kGatedWarps, k));
}

int gated_segments(int L) { return (L + kGatedCkpt - 1) / kGatedCkpt; }

void gated_plan(int B, int L, int D, bool backward, int sms, GatedParams* p) {
  const int ts = backward ? kGatedBwdSteps : kGatedFwdSteps, segs = (L + ts - 1) / ts;
  const long long wave = (backward ? 16LL : 24LL) * sms;    // warps that are resident
  const long long tiles64 = (D + 63) / 64;
  p->lanes = 32;
  p->splits = 1;
  p->solo = !backward && tiles64 * B >= wave;
  if (p->solo) {                                            // a row per warp
    p->warps = 4;
    p->rows = B / 4 + (B % 4 != 0) < 65535 ? (B + 3) / 4 : 65535;
    return;
  }
  // few warps per CTA while rows are many: 256 x 64 x 2048 bf16 backward 111 us at two,
  // 118 at four, 127 at eight
  int warps = 2;
  while (warps < kGatedWarps && tiles64 * B * warps * 2 <= wave) warps *= 2;
  if (warps > segs) warps = segs;
  p->warps = warps;
  const long long slots = wave / warps;
  // Of the tile widths and time splits whose every CTA has a pass of its own, the one
  // with most CTAs in one wave; wide tiles and few splits among equals.  A cluster lies in
  // one group of SMs, so fewer CTAs are resident in clusters (1 x 12523 x 3592 bf16: 57
  // clusters of 7, of which 56 are resident, 178 us, of 6 142; 2 x 16001 x 1280 fp32
  // backward: 40 of 7, of which 37 are, 288, of 6 200).  Measured: 1 x 16384 x 1024 bf16 128
  // CTAs of tile 64 93 us, 256 of 32 49, 384 of 16 49.
  auto tiles = [&](int l) { return (long long)(D + 2 * l - 1) / (2 * l); };
  long long most = tiles(32) * B;
  for (int l = 32; l >= 8; l /= 2)
    for (int k = 1; k <= 8; ++k) {
      const long long ctas = tiles(l) * B * k;
      if (ctas > slots || ctas <= most || segs < (long long)k * warps * (32 / l)) continue;
      if (k == 1 || (warps == kGatedWarps &&
                     ctas <= (backward ? gated_bwd_in_clusters(k) : fwd_in_clusters(k)))) {
        most = ctas;
        p->lanes = l;
        p->splits = k;
      }
    }
  long long gy = B, cap = slots / (tiles(p->lanes) * p->splits);
  if (cap < 1) cap = 1;
  if (cap > 65535) cap = 65535;
  if (gy > cap) {
    const long long each = (B + cap - 1) / cap;            // rows of a CTA, of equal number
    gy = (B + each - 1) / each;
  }
  p->rows = (int)gy;
}

cudaError_t launch_gated_fwd(const GatedParams& p, cudaStream_t s) {
  if (p.dtype == M3_F32)
    return p.copy == kVectors ? fwd_lanes<float, kVectors>(p, s) : fwd_lanes<float, kWords>(p, s);
  using B = __nv_bfloat16;
  return p.copy == kVectors ? fwd_lanes<B, kVectors>(p, s)
         : p.copy == kWords ? fwd_lanes<B, kWords>(p, s)
                            : fwd_lanes<B, kAny>(p, s);
}

cudaError_t launch_gated_step(const GatedStepParams& p, cudaStream_t s) {
  const int e = dsize(p.dtype);
  auto ok = [&](int v) {
    const int b = v * e < 16 ? v * e : 16;
    return p.D % v == 0 && p.ld_x % v == 0 && p.ld_r % v == 0 && p.ld_i % v == 0 &&
           aligned(p.h, 16) && aligned(p.x, b) && aligned(p.rg, b) && aligned(p.ig, b) &&
           aligned(p.y, b);
  };
  // 4 channels per thread: 8 of bf16 took 4.8 us instead of 3.8 for 100 rows of 4000,
  // 14.4 instead of 14.0 for 2048 of 2048
  if (p.dtype == M3_BF16)
    return ok(4) ? step_impl<__nv_bfloat16, 4>(p, s) : step_impl<__nv_bfloat16, 1>(p, s);
  return ok(4) ? step_impl<float, 4>(p, s) : step_impl<float, 1>(p, s);
}

}  // namespace m3
