// Selective scan, one token per row (the recurrence stands in
// m3_selective.cuh), in place on the state h (B, D, N).
//
// Bound by memory: the state is read and written once, 8 bytes per state and
// row against a few bytes per channel for everything else.  A lane group owns
// one channel, four states per thread, for kRows rows at a time: kRows
// independent 16-byte loads are in flight per thread, A is read once for all of
// them, and the rows' step sizes and outputs are spread over the group's lanes
// (each lane evaluates softplus and silu for its own rows and hands the step
// size to the others by shuffles).  2048 rows, D = 1024, N = 32, bf16: 94 us,
// 5.9 TB/s; 124 us with predicates and addresses per row and state.  fp32: 105 us
// (some of B and C in local memory at the 80 registers of six CTAs per SM).
#include "m3_api_util.h"
#include "m3_selective.cuh"

namespace m3 {
namespace {

constexpr int kRows = 8, kHalf = 4;

// FULL: all kRows rows and all states of the lane exist (no predicates; they and
// the addresses cost more than the recurrence otherwise).
template <typename T, int LN, bool VEC, bool FULL>
__device__ __forceinline__ void step_rows(const SelStepParams& p, int q, int d, size_t b0,
                                          int rows) {
  constexpr int KR = LN <= kRows ? kRows / LN : 1;   // rows per lane
  constexpr int PR = LN <= kRows ? 1 : LN / kRows;   // lanes per row
  const int n0 = 4 * q;
  const bool live = FULL || d < p.D, has = FULL || (live && n0 < p.N);
  float* const hp = p.h + (b0 * p.D + d) * p.N + n0;
  const size_t hs = (size_t)p.D * p.N;
  float4 h[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    h[r] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (FULL || (has && r < rows)) {
      if (VEC) h[r] = *reinterpret_cast<const float4*>(hp + r * hs);
      else h[r] = load_quad_any(p.h, b0 + r, d, n0, p.D, p.N);
    }
  }
  // the lane's own rows: q / PR * KR + i
  const float bias = (live && p.dt_bias) ? p.dt_bias[d] : 0.f;
  const float dsk = (live && p.dskip) ? p.dskip[d] : 0.f;
  float de[KR], uu[KR], zz[KR];
#pragma unroll
  for (int i = 0; i < KR; ++i) {
    const int r = q / PR * KR + i;
    de[i] = uu[i] = zz[i] = 0.f;
    if (FULL || (live && r < rows)) {
      const size_t b = b0 + r;
      uu[i] = Elem<T>::get(static_cast<const T*>(p.u)[b * p.ld_u + d]);
      de[i] = Elem<T>::get(static_cast<const T*>(p.dt)[b * p.ld_dt + d]) + bias;
      if (p.z) zz[i] = Elem<T>::get(static_cast<const T*>(p.z)[b * p.ld_z + d]);
    }
  }
  float4 a2 = make_float4(0.f, 0.f, 0.f, 0.f);
  if (has)
    a2 = VEC ? *reinterpret_cast<const float4*>(p.A + (size_t)d * p.N + n0)
             : load_quad_any(p.A, 0, d, n0, p.D, p.N);
  a2 = powers_of(a2);
#pragma unroll
  for (int i = 0; i < KR; ++i)
    if (FULL || (live && q / PR * KR + i < rows)) de[i] = step_size(de[i], p.softplus);
  const T* const pb = static_cast<const T*>(p.Bm) + b0 * p.ld_b + n0;
  const T* const pc = static_cast<const T*>(p.Cm) + b0 * p.ld_c + n0;
  float y[kRows];
#pragma unroll
  for (int r0 = 0; r0 < kRows; r0 += kHalf) {
    // the rows' B and C together, ahead of the stores that the loads could not pass
    Pack<T, 4> bv[kHalf], cv[kHalf];
#pragma unroll
    for (int i = 0; i < kHalf; ++i) {
      const int r = r0 + i;
      if (!FULL) {
        bv[i].zero();
        cv[i].zero();
      }
      if (FULL || (has && r < rows)) {
        if (VEC) {
          bv[i] = ld_pack<T, 4>(pb + r * p.ld_b);
          cv[i] = ld_pack<T, 4>(pc + r * p.ld_c);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (n0 + j < p.N) {
              bv[i].load_one(j, pb + r * p.ld_b);
              cv[i].load_one(j, pc + r * p.ld_c);
            }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kHalf; ++i) {
      const int r = r0 + i, src = r / KR * PR;
      const float der = __shfl_sync(0xffffffffu, de[r % KR], src, LN);
      const float dur = der * __shfl_sync(0xffffffffu, uu[r % KR], src, LN);
      h[r].x = fmaf(ex2_approx(fmaf(der, a2.x, kGateShift)), h[r].x, dur * bv[i].get(0));
      h[r].y = fmaf(ex2_approx(fmaf(der, a2.y, kGateShift)), h[r].y, dur * bv[i].get(1));
      h[r].z = fmaf(ex2_approx(fmaf(der, a2.z, kGateShift)), h[r].z, dur * bv[i].get(2));
      h[r].w = fmaf(ex2_approx(fmaf(der, a2.w, kGateShift)), h[r].w, dur * bv[i].get(3));
      y[r] = fmaf(h[r].x, cv[i].get(0), h[r].y * cv[i].get(1)) +
             fmaf(h[r].z, cv[i].get(2), h[r].w * cv[i].get(3));
      if (FULL || (has && r < rows)) {
        if (VEC) *reinterpret_cast<float4*>(hp + r * hs) = h[r];
        else store_quad_any(h[r], p.h, b0 + r, d, n0, p.D, p.N);
      }
    }
  }
  lane_sum<kRows, LN>(y, q);   // the lane's own rows
  if (live && q % PR == 0)
#pragma unroll
    for (int i = 0; i < KR; ++i) {
      const int r = q / PR * KR + i;
      if (FULL || r < rows) {
        float v = fmaf(dsk, uu[i], y[i]);
        if (p.z) v *= silu_f(zz[i]);
        static_cast<T*>(p.y)[(b0 + r) * p.D + d] = Elem<T>::put(v);
      }
    }
}

template <typename T, int LN, bool VEC>
__global__ void __launch_bounds__(128, 6) sel_step_kernel(const SelStepParams p) {
  constexpr int CH = 128 / LN;   // channels per CTA
  const int q = threadIdx.x % LN, d = (int)(blockIdx.x * CH + threadIdx.x / LN);
  const size_t b0 = (size_t)blockIdx.y * kRows;
  const int rows = (int)min((size_t)kRows, (size_t)p.B - b0);
  if (VEC && rows == kRows && p.N == 4 * LN && (int)(blockIdx.x + 1) * CH <= p.D)
    step_rows<T, LN, VEC, true>(p, q, d, b0, rows);
  else
    step_rows<T, LN, VEC, false>(p, q, d, b0, rows);
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
  const bool vec = p.N % 4 == 0 && aligned(p.h, 16) && aligned(p.A, 16) && aligned(p.Bm, a) && aligned(p.Cm, a) &&
                   p.ld_b % 4 == 0 && p.ld_c % 4 == 0;
  return p.dtype == M3_BF16 ? step_lanes<__nv_bfloat16>(p, vec, s) : step_lanes<float>(p, vec, s);
}

}  // namespace m3
