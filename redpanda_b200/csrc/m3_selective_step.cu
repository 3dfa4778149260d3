// Selective scan, one token per row (the recurrence stands in
// m3_selective.cuh), in place on the state h (B, D, N).
//
// Bound by memory: the state is read and written once, 8 bytes per state and
// row against a few bytes per channel for everything else.  A lane group owns
// one channel, four states per thread, for kRows rows at a time: kRows
// independent 16-byte loads are in flight per thread, A is read once for all of
// them, and the rows' step sizes and outputs are spread over the group's lanes
// (each lane evaluates softplus and silu for its own rows and hands the step
// size to the others by shuffles).
#include "m3_api_util.h"
#include "m3_selective.cuh"

namespace m3 {
namespace {

constexpr int kRows = 8;

template <typename T, int LN, bool VEC>
__global__ void __launch_bounds__(128) sel_step_kernel(const SelStepParams p) {
  constexpr int KR = LN <= kRows ? kRows / LN : 1;   // rows per lane
  constexpr int PR = LN <= kRows ? 1 : LN / kRows;   // lanes per row
  const int q = threadIdx.x % LN, d = (int)(blockIdx.x * (128 / LN) + threadIdx.x / LN);
  const int n0 = 4 * q;
  const size_t b0 = (size_t)blockIdx.y * kRows;
  const int rows = (int)min((size_t)kRows, (size_t)p.B - b0);
  const bool live = d < p.D;
  const bool has = live && n0 < p.N;

  float4 h[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    h[r] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (has && r < rows) {
      const float* src = p.h + ((b0 + r) * p.D + d) * p.N + n0;
      if (VEC) h[r] = *reinterpret_cast<const float4*>(src);
      else {
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = n0 + j < p.N ? src[j] : 0.f;
        h[r] = make_float4(v[0], v[1], v[2], v[3]);
      }
    }
  }
  float a2[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    a2[j] = (has && n0 + j < p.N) ? p.A[(size_t)d * p.N + n0 + j] * kLog2e : 0.f;
  // the lane's own rows: q / PR * KR + i
  const float bias = (live && p.dt_bias) ? p.dt_bias[d] : 0.f;
  const float dsk = (live && p.dskip) ? p.dskip[d] : 0.f;
  float de[KR], uu[KR], zz[KR];
#pragma unroll
  for (int i = 0; i < KR; ++i) {
    const int r = q / PR * KR + i;
    de[i] = uu[i] = zz[i] = 0.f;
    if (live && r < rows) {
      const size_t b = b0 + r;
      uu[i] = Elem<T>::get(static_cast<const T*>(p.u)[b * p.ld_u + d]);
      de[i] = step_size(Elem<T>::get(static_cast<const T*>(p.dt)[b * p.ld_dt + d]) + bias,
                        p.softplus);
      if (p.z) zz[i] = Elem<T>::get(static_cast<const T*>(p.z)[b * p.ld_z + d]);
    }
  }
  float y[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int src = r / KR * PR;
    const float der = __shfl_sync(0xffffffffu, de[r % KR], src, LN);
    const float dur = der * __shfl_sync(0xffffffffu, uu[r % KR], src, LN);
    Pack<T, 4> bv = zero_pack<T, 4>(), cv = zero_pack<T, 4>();
    if (has && r < rows) {
      const T* pb = static_cast<const T*>(p.Bm) + (b0 + r) * p.ld_b + n0;
      const T* pc = static_cast<const T*>(p.Cm) + (b0 + r) * p.ld_c + n0;
      if (VEC) {
        bv = ld_pack<T, 4>(pb);
        cv = ld_pack<T, 4>(pc);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n0 + j < p.N) {
            bv.load_one(j, pb);
            cv.load_one(j, pc);
          }
      }
    }
    h[r].x = fmaf(ex2_approx(der * a2[0]), h[r].x, dur * bv.get(0));
    h[r].y = fmaf(ex2_approx(der * a2[1]), h[r].y, dur * bv.get(1));
    h[r].z = fmaf(ex2_approx(der * a2[2]), h[r].z, dur * bv.get(2));
    h[r].w = fmaf(ex2_approx(der * a2[3]), h[r].w, dur * bv.get(3));
    y[r] = fmaf(h[r].x, cv.get(0), h[r].y * cv.get(1)) +
           fmaf(h[r].z, cv.get(2), h[r].w * cv.get(3));
    if (has && r < rows) {
      float* dst = p.h + ((b0 + r) * p.D + d) * p.N + n0;
      if (VEC) *reinterpret_cast<float4*>(dst) = h[r];
      else {
        const float v[4] = {h[r].x, h[r].y, h[r].z, h[r].w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n0 + j < p.N) dst[j] = v[j];
      }
    }
  }
  lane_sum<kRows, LN>(y, q);   // the lane's own rows
  if (live && q % PR == 0)
#pragma unroll
    for (int i = 0; i < KR; ++i) {
      const int r = q / PR * KR + i;
      if (r < rows) {
        float v = fmaf(dsk, uu[i], y[i]);
        if (p.z) v *= silu_f(zz[i]);
        static_cast<T*>(p.y)[(b0 + r) * p.D + d] = Elem<T>::put(v);
      }
    }
}

template <typename T, int LN>
cudaError_t step_typed(const SelStepParams& p, bool vec, cudaStream_t s) {
  const int per = 128 / LN;
  const dim3 grid((unsigned)((p.D + per - 1) / per), (unsigned)((p.B + kRows - 1) / kRows));
  if (vec) sel_step_kernel<T, LN, true><<<grid, 128, 0, s>>>(p);
  else sel_step_kernel<T, LN, false><<<grid, 128, 0, s>>>(p);
  return cudaGetLastError();
}

template <typename T>
cudaError_t step_lanes(const SelStepParams& p, bool vec, cudaStream_t s) {
  switch (sel_lanes(p.N)) {
    case 2: return step_typed<T, 2>(p, vec, s);
    case 4: return step_typed<T, 4>(p, vec, s);
    case 8: return step_typed<T, 8>(p, vec, s);
    case 16: return step_typed<T, 16>(p, vec, s);
    default: return step_typed<T, 32>(p, vec, s);
  }
}

}  // namespace

cudaError_t launch_sel_step(const SelStepParams& p, cudaStream_t s) {
  const int a = 4 * dsize(p.dtype);
  const bool vec = p.N % 4 == 0 && aligned(p.h, 16) && aligned(p.Bm, a) && aligned(p.Cm, a) &&
                   p.ld_b % 4 == 0 && p.ld_c % 4 == 0;
  return p.dtype == M3_BF16 ? step_lanes<__nv_bfloat16>(p, vec, s) : step_lanes<float>(p, vec, s);
}

}  // namespace m3
