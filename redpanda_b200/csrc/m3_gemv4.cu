// Product of at most 8 rows with weights of 4 bits and a scale per group of
// columns, with the element-wise work of m3_rows_linear around it (m3_gemv.cu):
//
//   w[o,k] = scale[o,k/G] (q[o,k] - 8) + center[o,k/G],  q in 0..15, G = 32, 64, 128
//   out = act(residual + (bias + n(x) w^T)),  n(x) = x or its RMS norm
//   sum_k x w = sum over groups of  scale sum x (q - 8) + center sum x
//
// Bound by the bytes of the codes for large weights (HBM, or L2 where they stay
// there) and by latency for small ones.  At one multiplication per weight and row
// the FMA pipe would be the limit from one row on (two instructions per weight to
// unpack, one per row), so the groups' sums run on the tensor cores (m16n8k16, the
// weights as the 16-row operand): q - 8 is exact in bf16, and an fp32 input is the
// sum of three bf16 numbers of 8 bits each, cut off its mantissa, so every product
// is exact; the parts of the rows take columns of their own (8 columns hold 8 rows of
// bf16, or 2 of fp32).  A group's sum is at most 8 instructions long and is folded
// into fp32 totals with its scale, so the tensor core's own accumulation, which
// cuts bits, is never long.  The norm's factor 1 / sqrt(mean(x^2) + eps) is a row's,
// and is applied to the total.
//
// A warp takes MT tiles of 16 outputs; the CTA's warps split tiles (mw) and the
// columns (kw), whose totals are added in order.  Codes are laid out once so that a
// lane's 16 bytes are its operand of four instructions (64 columns).  Inputs are
// staged in shared memory as the instruction's fragments, `chunk` columns at a time.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "m3_api_util.h"
#include "m3_ops.h"
#include "m3_pdl.cuh"
#include "m3_vec.cuh"

namespace m3 {
namespace {

constexpr int kAhead = 4;          // blocks of 64 columns in flight per warp

__device__ __forceinline__ void mma16816(float (&d)[4], const unsigned (&a)[4], unsigned b0,
                                         unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four pairs of codes as bf16 pairs of q - 8: the code in the low mantissa bits of
// 128 is 128 + q, and 128 + q - 136 is exact.
__device__ __forceinline__ void unpack(unsigned w, unsigned (&a)[4]) {
  const __nv_bfloat162 off = __halves2bfloat162(__ushort_as_bfloat16(0x4308),
                                                __ushort_as_bfloat16(0x4308));
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    unsigned v;
    asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;" : "=r"(v) : "r"(w >> (4 * r)));
    __nv_bfloat162 h = *reinterpret_cast<__nv_bfloat162*>(&v);
    h = __hsub2(h, off);
    a[r] = *reinterpret_cast<unsigned*>(&h);
  }
}

template <typename T>
__device__ __forceinline__ float2 load2(const T* p, int left, bool vec) {
  if (vec && left > 1) {
    const Pack<T, 2> v = ld_pack<T, 2>(p);
    return make_float2(v.get(0), v.get(1));
  }
  return make_float2(left > 0 ? Elem<T>::get(p[0]) : 0.f, left > 1 ? Elem<T>::get(p[1]) : 0.f);
}

__device__ __forceinline__ float warp_total(float v, int width) {
  for (int m = width / 2; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}

// the top 16 bits of a pair, x in the low half
__device__ __forceinline__ unsigned top_halves(float2 v) {
  return __byte_perm(__float_as_uint(v.x), __float_as_uint(v.y), 0x7632);
}
__device__ __forceinline__ float below(float v) {   // v without its top 16 bits (0 for infinity)
  const float t = __uint_as_float(__float_as_uint(v) & 0xffff0000u);
  return t == v ? 0.f : v - t;
}

// Stages the columns from k0 of every row: fragments, the groups' sums of the
// inputs and the squares' sums of every unit of U columns.
template <typename T, int NB, int G, bool CENTER>
__device__ void stage(const RowsQ4Params& p, int k0, int units, unsigned* frag, float* xs,
                      float* sq, int parts) {
  constexpr int U = G > 64 ? G : 64;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const T* x = static_cast<const T*>(p.x);
  for (int u = warp; u < units; u += warps) {
    for (int r = 0; r < p.rows; ++r) {
      float sum = 0.f, ss = 0.f;
#pragma unroll
      for (int h = 0; h < U / 64; ++h) {
        const int in = u * U + h * 64 + 2 * lane, k = k0 + in, left = p.d_in - k;
        float2 v = load2(x + (size_t)r * p.ld_x + (left > 0 ? k : 0), left, p.vec != 0);
        if (p.norm_w != nullptr) {
          ss = fmaf(v.x, v.x, fmaf(v.y, v.y, ss));
          const float2 w = load2(p.norm_w + (left > 0 ? k : 0), left, p.vec != 0);
          v.x *= w.x;
          v.y *= w.y;
        }
        if (CENTER) sum += v.x + v.y;
        // instruction k / 16; pairs t and (half) t + 4 of its 16 columns
        const int ks = in >> 4, half = lane >> 2 & 1, t = lane & 3;
        for (int s = 0; s < parts; ++s) {
          const int col = s * p.rows + r;
          frag[(((ks >> 1) * NB + (col >> 3)) * 32 + (col & 7) * 4 + t) * 4 + (ks & 1) * 2 + half] =
              top_halves(v);
          if (s + 1 < parts) v = make_float2(below(v.x), below(v.y));
        }
      }
      if (CENTER) {
        sum = warp_total(sum, G < 64 ? 16 : 32);
        if (G < 64 ? (lane & 15) == 0 : lane == 0)
          xs[(G < 64 ? u * 2 + (lane >> 4) : u) * (8 * NB) + r] = sum;
      }
      if (p.norm_w != nullptr) {
        ss = warp_total(ss, 32);
        if (lane == 0) sq[(k0 / U + u) * kQ4Rows + r] = ss;
      }
    }
  }
}

// shared memory: fragments, then the groups' sums, then the squares' sums of all units
struct Layout {
  int xs, sq, total;               // bytes
};
__host__ __device__ inline Layout layout(int NB, int G, bool center, int chunk, int units,
                                         bool norm) {
  Layout l;
  l.xs = chunk * 16 * NB;
  l.sq = l.xs + (center ? chunk / G * 8 * NB * 4 : 0);
  l.total = l.sq + (norm ? units * kQ4Rows * 4 : 0);
  return l;
}

template <typename T, int NB, int MT, int G, bool CENTER>
__global__ void __launch_bounds__(256, 2) rows_q4_kernel(const RowsQ4Params p) {
  constexpr int U = G > 64 ? G : 64, BU = U / 64, GU = U / G;   // a unit's columns, blocks, groups
  constexpr int NU = kAhead / BU / MT < 1 ? 1 : kAhead / BU / MT;   // units of a batch
  extern __shared__ __align__(16) char smem[];
  __shared__ float s_rstd[kQ4Rows];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int mw = warp % p.mw, kw = warp / p.mw;
  const int units = (p.d_in + U - 1) / U, per = (units + p.kw - 1) / p.kw;
  const int chunk_units = p.chunk / U, per_chunk = chunk_units / p.kw;
  const Layout lay = layout(NB, G, CENTER, p.chunk, units, p.norm_w != nullptr);
  unsigned* frag = reinterpret_cast<unsigned*>(smem);
  float* xs = reinterpret_cast<float*>(smem + lay.xs);
  float* sq = reinterpret_cast<float*>(smem + lay.sq);
  const int parts = sizeof(T) == 4 || p.norm_w != nullptr ? 3 : 1;
  const int tiles = (p.d_out + 15) / 16;
  const int tile0 = (blockIdx.x * p.mw + mw) * MT;
  pdl_launch_dependents();

  uint4 w[MT][NU][BU];
  uint2 sc[MT][NU][GU];
  auto load = [&](int i0) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NU; ++n) {
        const int u = (i0 + n) * p.kw + kw;
        const bool ok = i0 + n < per && u < units && tile0 + m < tiles;
#pragma unroll
        for (int b = 0; b < BU; ++b)
          w[m][n][b] = ok ? __ldg(p.codes + ((size_t)(tile0 + m) * units * BU + u * BU + b) * 32 +
                                  lane)
                          : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int g = 0; g < GU; ++g) {
          const size_t at = ((size_t)(tile0 + m) * units * GU + u * GU + g) * 8 + (lane >> 2);
          sc[m][n][g] = make_uint2(0, 0);
          if (ok) {
            if (CENTER) sc[m][n][g] = __ldg(static_cast<const uint2*>(p.scales) + at);
            else sc[m][n][g].x = __ldg(static_cast<const unsigned*>(p.scales) + at);
          }
        }
      }
  };
  load(0);
  pdl_wait();
  if (CENTER)   // the columns of the inputs' lower parts have no sum of their own
    for (int i = threadIdx.x; i < p.chunk / G * 8 * NB; i += blockDim.x) xs[i] = 0.f;

  float tot[MT][NB][4] = {};
  for (int i0 = 0; i0 < per; i0 += NU) {
    const int in = i0 % per_chunk;
    if (in == 0) {
      const int u0 = i0 * p.kw;
      __syncthreads();
      stage<T, NB, G, CENTER>(p, u0 * U, min(chunk_units, units - u0), frag, xs, sq, parts);
      __syncthreads();
    }
    uint4 cw[MT][NU][BU];
    uint2 cs[MT][NU][GU];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NU; ++n) {
#pragma unroll
        for (int b = 0; b < BU; ++b) cw[m][n][b] = w[m][n][b];
#pragma unroll
        for (int g = 0; g < GU; ++g) cs[m][n][g] = sc[m][n][g];
      }
    load(i0 + NU);
#pragma unroll
    for (int n = 0; n < NU; ++n) {
      const int u = (in + n) * p.kw + kw;            // in the chunk
      if (i0 + n >= per || (i0 + n) * p.kw + kw >= units) break;
      float acc[MT][NB][4];
#pragma unroll
      for (int b = 0; b < BU; ++b)
#pragma unroll
        for (int jp = 0; jp < 2; ++jp) {             // two instructions' worth of columns
          const bool first = G < 64 || (b == 0 && jp == 0), last = G < 64 || (b == BU - 1 && jp == 1);
          uint4 f[NB];
#pragma unroll
          for (int c = 0; c < NB; ++c)
            f[c] = *reinterpret_cast<const uint4*>(
                frag + (((u * (U / 32) + b * 2 + jp) * NB + c) * 32 + lane) * 4);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            if (first)
#pragma unroll
              for (int c = 0; c < NB; ++c)
                acc[m][c][0] = acc[m][c][1] = acc[m][c][2] = acc[m][c][3] = 0.f;
            unsigned a[4];
            unpack(jp ? cw[m][n][b].z : cw[m][n][b].x, a);
#pragma unroll
            for (int c = 0; c < NB; ++c) mma16816(acc[m][c], a, f[c].x, f[c].y);
            unpack(jp ? cw[m][n][b].w : cw[m][n][b].y, a);
#pragma unroll
            for (int c = 0; c < NB; ++c) mma16816(acc[m][c], a, f[c].z, f[c].w);
            if (last) {
              const uint2 s2 = cs[m][n][G < 64 ? jp : 0];
              float s0, s1, c0 = 0.f, c1 = 0.f;      // of outputs lane / 4 and lane / 4 + 8
              if (CENTER) {
                s0 = __uint_as_float(s2.x << 16);
                c0 = __uint_as_float(s2.x & 0xffff0000u);
                s1 = __uint_as_float(s2.y << 16);
                c1 = __uint_as_float(s2.y & 0xffff0000u);
              } else {
                s0 = __uint_as_float(s2.x << 16);
                s1 = __uint_as_float(s2.x & 0xffff0000u);
              }
#pragma unroll
              for (int c = 0; c < NB; ++c) {
                tot[m][c][0] = fmaf(s0, acc[m][c][0], tot[m][c][0]);
                tot[m][c][1] = fmaf(s0, acc[m][c][1], tot[m][c][1]);
                tot[m][c][2] = fmaf(s1, acc[m][c][2], tot[m][c][2]);
                tot[m][c][3] = fmaf(s1, acc[m][c][3], tot[m][c][3]);
                if (CENTER) {
                  const float2 v = *reinterpret_cast<const float2*>(
                      xs + (u * GU + (G < 64 ? jp : 0)) * (8 * NB) + c * 8 + 2 * (lane & 3));
                  tot[m][c][0] = fmaf(c0, v.x, tot[m][c][0]);
                  tot[m][c][1] = fmaf(c0, v.y, tot[m][c][1]);
                  tot[m][c][2] = fmaf(c1, v.x, tot[m][c][2]);
                  tot[m][c][3] = fmaf(c1, v.y, tot[m][c][3]);
                }
              }
            }
          }
        }
    }
  }

  // the rows' 1 / sqrt(mean(x^2) + eps): units in order, strided over a warp's lanes
  if (p.norm_w != nullptr)
    for (int r = warp; r < p.rows; r += blockDim.x >> 5) {
      float v = 0.f;
      for (int u = lane; u < units; u += 32) v += sq[u * kQ4Rows + r];
      v = warp_total(v, 32);
      if (lane == 0) s_rstd[r] = rsqrtf(v / (float)p.d_in + p.eps);
    }
  __syncthreads();
  // totals of every warp: (kw, outputs of the CTA, columns)
  float* red = reinterpret_cast<float*>(smem);
  const int outs = 16 * MT * p.mw;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int c = 0; c < NB; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int o = (mw * MT + m) * 16 + (lane >> 2) + (i >> 1) * 8;
        red[((size_t)kw * outs + o) * (8 * NB) + c * 8 + 2 * (lane & 3) + (i & 1)] = tot[m][c][i];
      }
  __syncthreads();
  for (int i = threadIdx.x; i < outs * p.rows; i += blockDim.x) {
    const int r = i / outs, o = i - r * outs, out = blockIdx.x * outs + o;
    if (out >= p.d_out) continue;
    float v = 0.f;
    for (int s = parts - 1; s >= 0; --s)             // the smallest part first
      for (int k = 0; k < p.kw; ++k) v += red[((size_t)k * outs + o) * (8 * NB) + s * p.rows + r];
    if (p.norm_w != nullptr) v *= s_rstd[r];
    if (p.bias != nullptr) v += p.bias[out];
    if (p.residual != nullptr)
      v += Elem<T>::get(static_cast<const T*>(p.residual)[(size_t)r * p.ld_r + out]);
    if (out < p.split) {
      if (p.silu) v = __fdiv_rn(v, 1.f + expf(-v));
      static_cast<T*>(p.out0)[(size_t)r * p.ld0 + out] = Elem<T>::put(v);
    } else {
      static_cast<T*>(p.out1)[(size_t)r * p.ld1 + (out - p.split)] = Elem<T>::put(v);
    }
  }
}

template <typename T, int NB, int MT, int G, bool CENTER>
cudaError_t launch(RowsQ4Params p, cudaStream_t s) {
  constexpr int U = G > 64 ? G : 64, BU = U / 64;
  constexpr int NU = kAhead / BU / MT < 1 ? 1 : kAhead / BU / MT;
  constexpr int kSmem = 112 << 10;                   // two CTAs per SM
  const int units = (p.d_in + U - 1) / U;
  const bool norm = p.norm_w != nullptr;
  // as many columns at a time as fit, a whole number of batches of every warp; at
  // kw = 1 and d_in = kQ4MaxIn one batch and the squares' sums take 45 KB
  auto bytes = [&](int chunk) { return layout(NB, G, CENTER, chunk, units, norm).total; };
  while (p.kw > 1 && bytes(p.kw * NU * U) > kSmem) --p.kw;
  const int step = p.kw * NU * U;
  int chunk = (units * U + step - 1) / step * step;
  while (chunk > step && bytes(chunk) > kSmem) chunk -= step;
  p.chunk = chunk;
  const int red = p.kw * 16 * MT * p.mw * 8 * NB * 4, smem = bytes(chunk) > red ? bytes(chunk) : red;
  const cudaError_t e = allow_smem<rows_q4_kernel<T, NB, MT, G, CENTER>>(kSmem);
  if (e != cudaSuccess) return e;
  const int grid = (p.d_out + 16 * MT * p.mw - 1) / (16 * MT * p.mw);
  return launch_maybe_pdl(p.pdl != 0, rows_q4_kernel<T, NB, MT, G, CENTER>, dim3(grid),
                          dim3(32 * p.mw * p.kw), smem, s, p);
}

template <typename T, int NB, int MT>
cudaError_t with_group(const RowsQ4Params& p, cudaStream_t s) {
  if (p.center) {
    if (p.group == 32) return launch<T, NB, MT, 32, true>(p, s);
    if (p.group == 64) return launch<T, NB, MT, 64, true>(p, s);
    return launch<T, NB, MT, 128, true>(p, s);
  }
  if (p.group == 32) return launch<T, NB, MT, 32, false>(p, s);
  if (p.group == 64) return launch<T, NB, MT, 64, false>(p, s);
  return launch<T, NB, MT, 128, false>(p, s);
}

template <typename T>
cudaError_t with_type(RowsQ4Params p, cudaStream_t s) {
  const int parts = sizeof(T) == 4 || p.norm_w != nullptr ? 3 : 1;
  const int nb = (p.rows * parts + 7) / 8, unit = p.group > 64 ? p.group : 64;
  const int units = (p.d_in + unit - 1) / unit;
  const long long tiles = (p.d_out + 15) / 16;
  // Warps along the columns while tiles are few, along the outputs where they fill
  // the GPU twice over: fewer copies of the inputs are staged.
  int mt = 1, mw = 1;
  if (tiles >= 4LL * p.sms) mt = 2;
  while (mw < 4 && tiles >= 4LL * p.sms * mt * mw) mw *= 2;
  p.mw = mw;
  p.kw = 8 / mw < units ? 8 / mw : units;
  switch (nb * 2 + (mt - 1)) {
    case 2: return with_group<T, 1, 1>(p, s);
    case 3: return with_group<T, 1, 2>(p, s);
    case 4: return with_group<T, 2, 1>(p, s);
    case 5: return with_group<T, 2, 2>(p, s);
    case 6: return with_group<T, 3, 1>(p, s);
    default: return with_group<T, 3, 2>(p, s);
  }
}

}  // namespace

cudaError_t launch_rows_q4(const RowsQ4Params& p, cudaStream_t s) {
  return p.dtype == M3_BF16 ? with_type<__nv_bfloat16>(p, s) : with_type<float>(p, s);
}

}  // namespace m3
