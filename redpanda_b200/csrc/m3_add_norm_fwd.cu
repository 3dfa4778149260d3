// The residual's addition and the RMS norm behind it, forward.
//
//   s = x + res, rounded to the stream's type;  r = 1 / sqrt(mean(s^2) + eps);  y = s r w
//
// The norm is that of s as stored, so that the backward, which reads s, has the
// forward's values.  Bound by memory: x and res in, s and y out.  Layout as in
// m3_norm.cu: a warp or a CTA per row, the row in registers between the sum and
// the output, the next row's loads ahead of the reduction, persistent CTAs.  131072 x
// 768, bf16 branch into an fp32 stream, bf16 y: 212 us (5.7 TB/s).  16384 x 4096 bf16 92 us,
// fp32 171 (5.8 and 6.3 TB/s); 4096 x 16384 88 and 188; 2048 x 32768, where a thread's 32
// elements and their next ones spill, 141 and 356.
#include "m3_add_norm.cuh"

namespace m3 {
namespace {

template <typename TX, typename TS, typename TY, int VEC, int NV, bool WARP, int MAXT, int MINB>
__global__ void __launch_bounds__(MAXT, MINB) add_norm_fwd_kernel(const AddNormParams p) {
  constexpr int E = VEC * NV;
  __shared__ float red[2][64];
  const int tpr = WARP ? 32 : blockDim.x, rpc = WARP ? MAXT / 32 : 1;
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x, d = p.d;
  int flip = 0;
  const TX* x = static_cast<const TX*>(p.x);
  const TS* res = static_cast<const TS*>(p.res);
  const long long step = (long long)gridDim.x * rpc;
  long long r = (long long)blockIdx.x * rpc + (WARP ? threadIdx.x >> 5 : 0);
  Row<TX, VEC, NV> nx;
  Row<TS, VEC, NV> nr;
  if (r < p.rows) {
    nx.load(x + (size_t)r * p.ld_x, d, t, tpr);
    nr.load(res + (size_t)r * p.ld_r, d, t, tpr);
  }
  float w[E];
  load_f32<VEC, NV>(w, p.w, d, t, tpr);
  const float inv_d = 1.f / (float)d;
  for (; r < p.rows; r += step) {
    float v[E], q[1] = {0.f};
    TS* sr = static_cast<TS*>(p.s) + (size_t)r * d;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * tpr + t) * VEC;
      Pack<TS, VEC> o;
      o.zero();
#pragma unroll
      for (int j = 0; j < VEC; ++j) o.put(j, nx.get(i * VEC + j) + nr.get(i * VEC + j));
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        v[i * VEC + j] = o.get(j);
        q[0] = fmaf(v[i * VEC + j], v[i * VEC + j], q[0]);
      }
      if (c < d) st_pack<TS, VEC>(sr + c, o);
    }
    if (r + step < p.rows) {
      nx.load(x + (size_t)(r + step) * p.ld_x, d, t, tpr);
      nr.load(res + (size_t)(r + step) * p.ld_r, d, t, tpr);
    }
    row_sum<WARP>(q, red, flip);
    const float rs = rsqrtf(q[0] * inv_d + p.eps);
    if (t == 0 && p.rstd != nullptr) p.rstd[r] = rs;
    TY* yr = static_cast<TY*>(p.y) + (size_t)r * d;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * tpr + t) * VEC;
      if (c < d) {
        Pack<TY, VEC> o;
#pragma unroll
        for (int j = 0; j < VEC; ++j) o.put(j, v[i * VEC + j] * rs * w[i * VEC + j]);
        st_pack<TY, VEC>(yr + c, o);
      }
    }
  }
}

template <typename TX, typename TS, typename TY>
struct Launch {
  static constexpr bool kWide = sizeof(TX) == 2 || sizeof(TS) == 2 || sizeof(TY) == 2;
  static constexpr bool kEven = true;
  static constexpr int kFrom = 2048;
  static constexpr bool kWarpRows = true;
  const AddNormParams& p;
  cudaStream_t s;
  template <int VEC, int NV, bool WARP, int MAXT, int MINB>
  cudaError_t operator()(int nt) {
    const int rpc = WARP ? MAXT / 32 : 1;
    const long long want = (p.rows + rpc - 1) / rpc;
    const int per = WARP ? MINB : add_resident<add_norm_fwd_kernel<TX, TS, TY, VEC, NV, WARP, MAXT, MINB>>(nt);
    if (per <= 0) return cudaErrorInvalidConfiguration;
    const long long cap = (long long)p.sms * per;
    const int grid = (int)(want < cap ? want : cap);
    add_norm_fwd_kernel<TX, TS, TY, VEC, NV, WARP, MAXT, MINB><<<grid, nt, 0, s>>>(p);
    return cudaGetLastError();
  }
};

}  // namespace

cudaError_t launch_add_norm_fwd(const AddNormParams& p, cudaStream_t s) {
  const int ex = dsize(p.dtype_x), es = dsize(p.dtype_s), ey = dsize(p.dtype_y);
  auto ok = [&](int v) {
    return p.d % v == 0 && rows_ok(p.x, p.ld_x, ex, v) && rows_ok(p.res, p.ld_r, es, v) &&
           rows_ok(p.s, p.d, es, v) && rows_ok(p.y, p.d, ey, v);
  };
  const int vec = ex + es + ey < 12 && ok(8) ? 8 : ok(4) ? 4 : ok(2) ? 2 : 1;
  return with_types(p.dtype_x, p.dtype_s, p.dtype_y, [&](auto tx, auto ts, auto ty) {
    return add_dispatch(p.d, vec, Launch<decltype(tx), decltype(ts), decltype(ty)>{p, s});
  });
}

}  // namespace m3
