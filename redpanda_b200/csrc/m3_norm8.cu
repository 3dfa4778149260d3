// The RMS norm, of x or of the residual stream s = x + res, in 8 bits with scales:
// rows for a projection whose operands are 8 bits wide.
//
//   y = s r w (m3_add_norm_fwd.cu) in fp32, not rounded in between
//   scale = max(max |y| / top, 2^-126) over a row or over `group` columns of it, to 2^-23
//   q = y / scale, to 2^-22, rounded to nearest even and held to [-top, top]
//
// top is 448 (e4m3) or 127 (int8).  The floor of the scale keeps the quotient
// finite where a group is zero or below what fp32 divides by.  A NaN in a group
// makes its scale NaN, so nothing that depends on it passes for a number.
// Bound by memory, then by instructions (66 % of the issue slots: unpacking, the
// group's maximum over lanes, conversion); layout as m3_norm.cu's forward.  16384 x 4096
// bf16 with the addition and groups of 128: 86 us (5.5 TB/s); 173 us with a division per
// element and 8 elements per thread.
#include <cuda_fp8.h>

#include "m3_add_norm.cuh"

namespace m3 {
namespace {

__device__ __forceinline__ float nan_max(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// Largest value over the threads of a row, as row_sum.
template <bool WARP>
__device__ __forceinline__ float row_max(float v, float (*red)[64], int& flip) {
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) v = nan_max(v, __shfl_xor_sync(0xffffffffu, v, m));
  if constexpr (!WARP) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, W = blockDim.x >> 5;
    float* r = red[flip];
    flip ^= 1;
    if (lane == 0) r[warp] = v;
    __syncthreads();
    v = lane < W ? r[lane] : 0.f;
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) v = nan_max(v, __shfl_xor_sync(0xffffffffu, v, m));
  }
  return v;
}

// Codes of VEC values, the first in the lowest byte; one instruction per pair for
// e4m3 (which holds the result to 448), one per value for int8.
template <bool E4M3, int VEC>
__device__ __forceinline__ void store8(unsigned char* p, const float (&v)[VEC]) {
  unsigned b[(VEC + 3) / 4] = {};
#pragma unroll
  for (int j = 0; j < VEC; j += 2) {
    unsigned two;
    if (E4M3) {
      two = __nv_cvt_float2_to_fp8x2(make_float2(v[j], VEC > 1 ? v[j + (VEC > 1)] : 0.f),
                                     __NV_SATFINITE, __NV_E4M3);
    } else {
      auto one = [](float x) {
        const int i = __float2int_rn(x);
        return (unsigned)(i < -127 ? -127 : i > 127 ? 127 : i) & 0xffu;
      };
      two = one(v[j]) | (VEC > 1 ? one(v[j + (VEC > 1)]) << 8 : 0u);
    }
    b[j / 4] |= two << (j % 4 * 8);
  }
  if constexpr (VEC == 8) *reinterpret_cast<uint2*>(p) = make_uint2(b[0], b[1]);
  else if constexpr (VEC == 4) *reinterpret_cast<unsigned*>(p) = b[0];
  else if constexpr (VEC == 2) *reinterpret_cast<unsigned short*>(p) = (unsigned short)b[0];
  else *p = (unsigned char)b[0];
}

template <typename TX, typename TS, bool E4M3, int VEC, int NV, bool WARP, int MAXT, int MINB>
__global__ void __launch_bounds__(MAXT, MINB) norm8_kernel(const Norm8Params p) {
  constexpr int E = VEC * NV;
  constexpr float kTop = E4M3 ? 448.f : 127.f;
  __shared__ float red[2][64];
  const int tpr = WARP ? 32 : blockDim.x, rpc = WARP ? MAXT / 32 : 1;
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x, d = p.d;
  int flip = 0;
  const TX* x = static_cast<const TX*>(p.x);
  const TS* res = static_cast<const TS*>(p.res);
  const bool add = res != nullptr;
  const long long step = (long long)gridDim.x * rpc;
  long long r = (long long)blockIdx.x * rpc + (WARP ? threadIdx.x >> 5 : 0);
  Row<TX, VEC, NV> nx;
  Row<TS, VEC, NV> nr;
  if (r < p.rows) {
    nx.load(x + (size_t)r * p.ld_x, d, t, tpr);
    if (add) nr.load(res + (size_t)r * p.ld_r, d, t, tpr);
  }
  float w[E];
  load_f32<VEC, NV>(w, p.w, d, t, tpr);
  const float inv_d = 1.f / (float)d;
  for (; r < p.rows; r += step) {
    float v[E], q[1] = {0.f};
#pragma unroll
    for (int k = 0; k < E; ++k) v[k] = nx.get(k);
    if (add) {
      TS* sr = static_cast<TS*>(p.s) + (size_t)r * d;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * tpr + t) * VEC;
        Pack<TS, VEC> o;
        o.zero();
#pragma unroll
        for (int j = 0; j < VEC; ++j) o.put(j, v[i * VEC + j] + nr.get(i * VEC + j));
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i * VEC + j] = o.get(j);
        if (c < d) st_pack<TS, VEC>(sr + c, o);
      }
    }
#pragma unroll
    for (int k = 0; k < E; ++k) q[0] = fmaf(v[k], v[k], q[0]);
    if (r + step < p.rows) {
      nx.load(x + (size_t)(r + step) * p.ld_x, d, t, tpr);
      if (add) nr.load(res + (size_t)(r + step) * p.ld_r, d, t, tpr);
    }
    row_sum<WARP>(q, red, flip);
    const float rs = rsqrtf(q[0] * inv_d + p.eps);
    float top[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      top[i] = 0.f;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int k = i * VEC + j;
        v[k] = v[k] * rs * w[k];
        top[i] = nan_max(top[i], fabsf(v[k]));
      }
    }
    if (p.group == 0) {
      float m = top[0];
#pragma unroll
      for (int i = 1; i < NV; ++i) m = nan_max(m, top[i]);
      m = row_max<WARP>(m, red, flip);
#pragma unroll
      for (int i = 0; i < NV; ++i) top[i] = m;
    } else if constexpr (VEC > 2) {
      // a group's columns lie in group / VEC neighbouring lanes
      const int span = p.group / VEC;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        for (int m = 1; m < span; m <<= 1)
          top[i] = nan_max(top[i], __shfl_xor_sync(0xffffffffu, top[i], m));
    }
    unsigned char* qr = p.q + (size_t)r * d;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * tpr + t) * VEC;
      // the quotient as a product with the scale's approximate reciprocal: the unit's
      // 2^-23 and a rounding of 2^-24, together below 2^-22 of the quotient, where a
      // division has 2^-24.  So a quotient that near to the border of two codes may get
      // either (173 against 129 us with 8 elements per thread).
      const float scale = nan_max(top[i] * (1.f / kTop), 0x1p-126f), inv = rcp_approx(scale);
      if (c < d) {
        float u[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) u[j] = v[i * VEC + j] * inv;
        store8<E4M3, VEC>(qr + c, u);
        if (p.group == 0) {
          if (c == 0) p.scale[r] = scale;
        } else if (c % p.group == 0) {
          p.scale[(size_t)r * (d / p.group) + c / p.group] = scale;
        }
      }
    }
  }
}

template <typename TX, typename TS>
struct Launch {
  static constexpr bool kWide = true, kWarpRows = true;
  static constexpr bool kEven = true;
  static constexpr int kFrom = 1024;
  const Norm8Params& p;
  cudaStream_t s;
  template <int VEC, int NV, bool WARP, int MAXT, int MINB>
  cudaError_t operator()(int nt) {
    const int rpc = WARP ? MAXT / 32 : 1;
    const long long want = (p.rows + rpc - 1) / rpc;
    auto go = [&](auto e4m3) -> cudaError_t {
      constexpr auto* kern = norm8_kernel<TX, TS, decltype(e4m3)::value, VEC, NV, WARP, MAXT, MINB>;
      const int per = WARP ? MINB : add_resident<kern>(nt);
      if (per <= 0) return cudaErrorInvalidConfiguration;
      const long long cap = (long long)p.sms * per;
      kern<<<(int)(want < cap ? want : cap), nt, 0, s>>>(p);
      return cudaGetLastError();
    };
    return p.e4m3 ? go(std::true_type()) : go(std::false_type());
  }
};

}  // namespace

cudaError_t launch_norm8(const Norm8Params& p, cudaStream_t s) {
  const int ex = dsize(p.dtype_x), es = dsize(p.dtype_s);
  auto ok = [&](int v) {
    return p.d % v == 0 && rows_ok(p.x, p.ld_x, ex, v) && rows_ok(p.res, p.ld_r, es, v) &&
           rows_ok(p.s, p.d, es, v) && aligned(p.q, v);
  };
  const int vec = ok(8) ? 8 : ok(4) ? 4 : ok(2) ? 2 : 1;
  if (p.group != 0 && vec < 4) return cudaErrorInvalidValue;   // refused by the entry
  return with_types(p.dtype_x, p.dtype_s, M3_F32, [&](auto tx, auto ts, auto) {
    return add_dispatch(p.d, vec, Launch<decltype(tx), decltype(ts)>{p, s});
  });
}

}  // namespace m3
