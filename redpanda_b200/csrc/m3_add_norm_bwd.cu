// The residual's addition and the RMS norm behind it, backward.
//
//   with sh = s r, q = gy w:  ds = gs + r (q - sh mean(q sh)),  dx = dres = ds,
//                             dw = sum over rows of gy sh
//
// Bound by memory: s, gy and gs in, ds out, in the branch's type too where that is
// another.  Layout as the norm's backward (m3_norm.cu): every row is read once, the
// weight gradient of a thread's columns stays in registers over its rows, each CTA
// writes one partial row of dw and a second launch adds them in a fixed order.  131072
// x 768, gradients of bf16 y and of an fp32 stream: 242 us (6.7 TB/s).  Past 2048 columns
// three rows, their next ones, the weight and its gradient fill a thread's 128 registers
// (fp32: 92 bytes spilled), so that 16 warps are all an SM holds: 16384 x 4096 bf16 116 us,
// fp32 212 (4.6 and 5.1 TB/s).  Past 8192 a thread of up to 1024 has 64 registers, and 250
// to 1700 bytes are spilled: 4096 x 16384 bf16 174 us, fp32 418; 2048 x 32768 490 and 1000.
#include "m3_add_norm.cuh"
#include "m3_pdl.cuh"

namespace m3 {
namespace {

constexpr int kRowsFrom = 2048;

template <typename TX, typename TS, typename TY, int VEC, int NV, bool WARP, int MAXT, int MINB>
__global__ void __launch_bounds__(MAXT, MINB) add_norm_bwd_kernel(const AddNormBwdParams p) {
  constexpr int E = VEC * NV;
  __shared__ float red[2][64];
  __shared__ float comb[WARP ? E * 32 : 1];   // the CTA's warps' partials
  const int tpr = WARP ? 32 : blockDim.x, rpc = WARP ? MAXT / 32 : 1;
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x, d = p.d;
  int flip = 0;
  const TS* sp = static_cast<const TS*>(p.s);
  const TY* gy = static_cast<const TY*>(p.gy);
  const TS* gs = static_cast<const TS*>(p.gs);
  float w[E], dw[E];
  const long long step = (long long)gridDim.x * rpc;
  long long r = (long long)blockIdx.x * rpc + (WARP ? threadIdx.x >> 5 : 0);
  Row<TS, VEC, NV> cs, ca;
  Row<TY, VEC, NV> cg;
#pragma unroll
  for (int i = 0; i < NV; ++i) ca.p[i].zero();
  if (r < p.rows) {
    cs.load(sp + (size_t)r * p.ld_s, d, t, tpr);
    cg.load(gy + (size_t)r * d, d, t, tpr);
    if (gs != nullptr) ca.load(gs + (size_t)r * d, d, t, tpr);
  }
  load_f32<VEC, NV>(w, p.w, d, t, tpr);
#pragma unroll
  for (int k = 0; k < E; ++k) dw[k] = 0.f;
  const float inv_d = 1.f / (float)d;
  for (; r < p.rows; r += step) {
    Row<TS, VEC, NV> ns, na;
    Row<TY, VEC, NV> ng;
#pragma unroll
    for (int i = 0; i < NV; ++i) na.p[i].zero();
    if (r + step < p.rows) {
      ns.load(sp + (size_t)(r + step) * p.ld_s, d, t, tpr);
      ng.load(gy + (size_t)(r + step) * d, d, t, tpr);
      if (gs != nullptr) na.load(gs + (size_t)(r + step) * d, d, t, tpr);
    }
    const float rs = p.rstd[r];
    float s[1] = {0.f};
#pragma unroll
    for (int k = 0; k < E; ++k) {   // a column past d has gy = 0 and w = 0
      const float sh = cs.get(k) * rs, gk = cg.get(k);
      s[0] = fmaf(gk * w[k], sh, s[0]);
      dw[k] = fmaf(gk, sh, dw[k]);
    }
    row_sum<WARP>(s, red, flip);
    const float mx = s[0] * inv_d;
    TS* o = static_cast<TS*>(p.ds) + (size_t)r * d;
    TX* ox = static_cast<TX*>(p.dx) + (size_t)r * d;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * tpr + t) * VEC;
      if (c < d) {
        Pack<TS, VEC> v;
        Pack<TX, VEC> vx;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const int k = i * VEC + j;
          const float sh = cs.get(k) * rs;
          const float g = fmaf(rs, fmaf(cg.get(k), w[k], -sh * mx), ca.get(k));
          v.put(j, g);
          vx.put(j, g);
        }
        st_pack<TS, VEC>(o + c, v);
        if (sizeof(TX) != sizeof(TS) && p.dx != nullptr) st_pack<TX, VEC>(ox + c, vx);
      }
    }
    cs = ns;
    cg = ng;
    ca = na;
  }
  pdl_launch_dependents();
  float* part = p.part + (size_t)blockIdx.x * d;
  if constexpr (WARP) {
    const int row = threadIdx.x >> 5;
    for (int k = 0; k < rpc; ++k) {   // warps add in order
      if (row == k)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          float* a = comb + e * 32 + t;
          *a = k ? *a + dw[e] : dw[e];
        }
      __syncthreads();
    }
    if (row != 0) return;
#pragma unroll
    for (int e = 0; e < E; ++e) dw[e] = comb[e * 32 + t];
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int c = ((e / VEC) * tpr + t) * VEC + e % VEC;
    if (c < d) part[c] = dw[e];
  }
}

template <typename TX, typename TS, typename TY>
struct Launch {
  static constexpr bool kWide = sizeof(TX) == 2 || sizeof(TS) == 2 || sizeof(TY) == 2;
  static constexpr bool kEven = true;
  static constexpr int kFrom = kRowsFrom;
  static constexpr bool kWarpRows = false;
  const AddNormBwdParams& p;
  cudaStream_t s;
  template <int VEC, int NV, bool WARP, int MAXT, int MINB>
  cudaError_t operator()(int nt) {
    const int ctas = add_norm_bwd_ctas(p.rows, p.d, p.sms);
    add_norm_bwd_kernel<TX, TS, TY, VEC, NV, WARP, MAXT, MINB><<<ctas, nt, 0, s>>>(p);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    return launch_norm_reduce(p.part, ctas, p.d, 1, p.dw, nullptr, s);
  }
};

}  // namespace

// 768 threads per SM at 80 registers, 512 at 128 where a thread holds 16 elements
int add_norm_bwd_ctas(long long rows, int d, int sms) {
  const int rpc = d <= 256 ? 4 : 1, nt = d <= 256 ? 128 : add_threads(d, kRowsFrom);
  const int per = d <= kRowsFrom ? 768 / nt : nt <= 512 ? 512 / nt : 1;
  const long long want = (rows + rpc - 1) / rpc, cap = (long long)sms * per;
  return (int)(want < cap ? want : cap);
}

cudaError_t launch_add_norm_bwd(const AddNormBwdParams& p, cudaStream_t s) {
  const int ex = dsize(p.dtype_x), es = dsize(p.dtype_s), ey = dsize(p.dtype_y);
  auto ok = [&](int v) {
    return p.d % v == 0 && rows_ok(p.s, p.ld_s, es, v) && rows_ok(p.gy, p.d, ey, v) &&
           rows_ok(p.gs, p.d, es, v) && rows_ok(p.ds, p.d, es, v) && rows_ok(p.dx, p.d, ex, v);
  };
  const int vec = ex + es + ey < 12 && ok(8) ? 8 : ok(4) ? 4 : ok(2) ? 2 : 1;
  return with_types(p.dtype_x, p.dtype_s, p.dtype_y, [&](auto tx, auto ts, auto ty) {
    return add_dispatch(p.d, vec, Launch<decltype(tx), decltype(ts), decltype(ty)>{p, s});
  });
}

}  // namespace m3
