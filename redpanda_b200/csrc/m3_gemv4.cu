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
// bf16, or 2 of fp32); the inputs' sums are a product with ones.  A group's sum is at
// most 8 instructions long and is folded into fp32 totals with its scale, so the tensor
// core's own accumulation, which cuts bits, is never long.  The norm's factor
// 1 / sqrt(mean(x^2) + eps) is a row's, and is applied to the total.
//
// A warp takes MT tiles of 16 outputs; the CTA's warps split tiles (mw) and the
// columns (kw), whose totals are added in order.  Codes are laid out once so that a
// lane's 16 bytes are its operand of four instructions (64 columns).  Inputs are
// staged in shared memory, `chunk` columns at a time; codes and scales come through a
// ring of asynchronous copies per warp.
//
// 3 rows of bf16, 8192 x 65536, groups of 128: 67 us (4.1 TB/s; the bytes take 42).  One
// wave of CTAs with these rings reads the codes alone in 55-62 us, whatever the rings'
// depth; many small CTAs read them in 43-45, but each would stage the inputs again.  8
// rows of fp32, 768 x 8192: 8.3 us.  1 row, 384 x 1536 with the norm and silu: 4.3 us.
// Many rows of fp32 over long inputs are bound by staging, which every CTA repeats: 8 rows,
// 8192 x 8192: 42 us for 38 MB; 2048 x 50304 with the norm: 49 us for 60 MB.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "m3_api_util.h"
#include "m3_ops.h"
#include "m3_pdl.cuh"
#include "m3_vec.cuh"

namespace m3 {
namespace {

constexpr int kPad = 32;           // columns behind a staged row
constexpr int kSquares = 128;      // columns of a sum of the norm's squares: a warp's at a time

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

// The inputs in shared memory: `cols` rows of bf16 (part by part, row by row), of the
// chunk's columns and 32 more (so that 8 lanes' 16 bytes lie in different banks).  The
// instruction's order of the 16 columns it takes at a time is free as long as both
// operands agree: lane l's two instructions of 32 columns take the 8 columns from
// 8 (l % 4), so its operands are 16 consecutive bytes of a row.
//
__device__ __forceinline__ float4 load4(const float* p, int left, bool vec) {
  if (vec && left >= 4) return *reinterpret_cast<const float4*>(p);
  return make_float4(left > 0 ? p[0] : 0.f, left > 1 ? p[1] : 0.f, left > 2 ? p[2] : 0.f,
                     left > 3 ? p[3] : 0.f);
}
// Element j of a row of which `left` are there (any address but the row's start is one of
// the row's own); the bits, so that a load's result is not used where it is asked for.
template <typename T>
__device__ __forceinline__ T element(const T* p, int j, int left) {
  return p[max(min(j, left - 1), 0)];
}
__device__ __forceinline__ uint2 top_halves(const float4& v) {
  return make_uint2(top_halves(make_float2(v.x, v.y)), top_halves(make_float2(v.z, v.w)));
}
__device__ __forceinline__ float4 below(const float4& v) {
  return make_float4(below(v.x), below(v.y), below(v.z), below(v.w));
}

// Sums of every row's value over the lanes of a warp: lane l has that of row
// l / (32 / R) (R rows, a power of two; 5 + R shuffles instead of 5 R).
template <int R>
__device__ __forceinline__ float row_totals(const float (&v)[kQ4Rows]) {
  const int lane = threadIdx.x & 31;
  float a[R];
#pragma unroll
  for (int r = 0; r < R; ++r) a[r] = v[r];
  int m = 16;
#pragma unroll
  for (int n = R / 2; n > 0; n >>= 1, m >>= 1)
#pragma unroll
    for (int r = 0; r < n; ++r) {
      const bool up = lane & m;
      const float keep = up ? a[r + n] : a[r], give = up ? a[r] : a[r + n];
      a[r] = keep + __shfl_xor_sync(0xffffffffu, give, m);
    }
  float t = a[0];
  for (; m > 0; m >>= 1) t += __shfl_xor_sync(0xffffffffu, t, m);
  return t;
}

// f(r, columns of row r) for every row of bf16, four columns from x, of which `left` are
// there; every load before any value is widened, four rows at a time where elements are
// loaded one by one (a value widened beside its load is waited for there: 4 rows with the
// norm, 4985 -> 1617 23 against 14 us).
template <typename T, typename F>
__device__ __forceinline__ void for_rows(const T* x, long long ld, int rows, int left, bool vec,
                                         F&& f) {
  if (__all_sync(0xffffffffu, vec && left >= 4)) {
    Pack<T, 4> v[kQ4Rows];
#pragma unroll
    for (int r = 0; r < kQ4Rows; ++r)
      if (r < rows) v[r] = ld_pack<T, 4>(x + r * ld);
#pragma unroll
    for (int r = 0; r < kQ4Rows; ++r) {
      if (r >= rows) break;
      f(r, make_float4(v[r].get(0), v[r].get(1), v[r].get(2), v[r].get(3)));
    }
  } else {
#pragma unroll
    for (int r0 = 0; r0 < kQ4Rows; r0 += 4) {
      T e[4][4];
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (r0 + r < rows)
#pragma unroll
          for (int j = 0; j < 4; ++j) e[r][j] = element(x + (r0 + r) * ld, j, left);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (r0 + r < rows) {
          auto get = [&](int j) { return j < left ? Elem<T>::get(e[r][j]) : 0.f; };
          f(r0 + r, make_float4(get(0), get(1), get(2), get(3)));
        }
    }
  }
}

// Stages the columns from k0 of every row, with the squares' sums of every 128 columns (k0
// is a multiple of 128 where there is a norm: each sum is written once).
// bf16 rows without a norm are copied as they are, 16 or 4 bytes at a time, or, where they
// start in the middle of a word, by elements (7 rows, 7050 -> 1299: by words 10 us, split
// as the others are 35).
template <typename T>
__device__ void stage(const RowsQ4Params& p, int k0, int n, char* rows, float* sq, int parts) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int row = (p.chunk + kPad) * 2;              // bytes
  const T* x = static_cast<const T*>(p.x) + k0;
  if constexpr (sizeof(T) == 2) {
    if (parts == 1 && p.vec8 == 2) {
      for (int r = 0; r < p.rows; ++r)
        for (int c = (warp * 32 + lane) * 8; c < n; c += warps * 256) {
          const int left = (p.d_in - k0 - c) * 2, bytes = left < 0 ? 0 : left < 16 ? left : 16;
          const T* from = x + (size_t)r * p.ld_x + (bytes > 0 ? c : 0);
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                           (unsigned)__cvta_generic_to_shared(rows + r * row + c * 2)),
                       "l"(from), "r"(bytes)
                       : "memory");
        }
      asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
      return;
    }
    if (parts == 1 && p.vec8 == 1) {
      for (int r = 0; r < p.rows; ++r)
        for (int c = (warp * 32 + lane) * 2; c < n; c += warps * 64) {
          const int left = (p.d_in - k0 - c) * 2, bytes = left < 0 ? 0 : left < 4 ? left : 4;
          const T* from = x + (size_t)r * p.ld_x + (bytes > 0 ? c : 0);
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(
                           (unsigned)__cvta_generic_to_shared(rows + r * row + c * 2)),
                       "l"(from), "r"(bytes)
                       : "memory");
        }
      asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
      return;
    }
    if (parts == 1) {
      for (int c0 = warp * 128; c0 < n; c0 += warps * 128) {
#pragma unroll
        for (int r0 = 0; r0 < kQ4Rows; r0 += 4) {
          unsigned short v[4][4];
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (r0 + r < p.rows)
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int c = c0 + lane + 32 * j;
                v[r][j] = reinterpret_cast<const unsigned short*>(x)[(r0 + r) * p.ld_x +
                                                                     (c < p.d_in - k0 ? c : 0)];
              }
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (r0 + r < p.rows)
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int c = c0 + lane + 32 * j;
                if (c < n)
                  *reinterpret_cast<unsigned short*>(rows + (r0 + r) * row + c * 2) =
                      c < p.d_in - k0 ? v[r][j] : (unsigned short)0;
              }
        }
      }
      return;
    }
  }
  const bool vec = p.vec != 0;
  for (int c0 = warp * 128; c0 < n; c0 += warps * 128) {
    const int c = c0 + lane * 4, left = p.d_in - k0 - c, at = left > 0 ? c : 0;
    float4 w;
    float ss[kQ4Rows] = {};
    auto split = [&](int r, float4 y) {
      if (p.norm_w != nullptr) {
        ss[r] = fmaf(y.x, y.x, y.y * y.y) + fmaf(y.z, y.z, y.w * y.w);
        y = make_float4(y.x * w.x, y.y * w.y, y.z * w.z, y.w * w.w);
      }
      if (c < n) {
        char* to = rows + r * row + c * 2;
        *reinterpret_cast<uint2*>(to) = top_halves(y);
        if (parts == 3) {
          y = below(y);
          *reinterpret_cast<uint2*>(to + p.rows * row) = top_halves(y);
          *reinterpret_cast<uint2*>(to + 2 * p.rows * row) = top_halves(below(y));
        }
      }
    };
    if constexpr (sizeof(T) == 4) {                  // every row's loads before any is used
      float4 v[kQ4Rows];
#pragma unroll
      for (int r = 0; r < kQ4Rows; ++r)
        if (r < p.rows) v[r] = load4(x + (size_t)r * p.ld_x + at, left, vec);
      if (p.norm_w != nullptr) w = load4(p.norm_w + k0 + at, left, vec);
#pragma unroll
      for (int r = 0; r < kQ4Rows; ++r) {
        if (r >= p.rows) break;
        split(r, v[r]);
      }
    } else {
      if (p.norm_w != nullptr) w = load4(p.norm_w + k0 + at, left, vec);
      for_rows(x + at, p.ld_x, p.rows, left, vec, split);
    }
    if (p.norm_w != nullptr) {
      float* to = sq + (k0 + c0) / kSquares * kQ4Rows;
      if (p.rows == 1) {
        const float t = row_totals<1>(ss);
        if (lane == 0) to[0] = t;
      } else {
        const float t = row_totals<8>(ss);
        if (lane % 4 == 0) to[lane / 4] = t;
      }
    }
  }
}

// A warp's ring of units in flight: MT tiles' codes, then their scales.
template <int MT, int G, bool CENTER>
struct Ring {
  static constexpr int U = G > 64 ? G : 64, BU = U / 64, GU = U / G;   // columns, blocks, groups
  static constexpr int kScale = GU * 8 * (CENTER ? 8 : 4);             // bytes per tile and unit
  static constexpr int kSlot = MT * (BU * 512 + kScale);
  static constexpr int kSlots = MT * BU == 1 ? 8 : MT * BU == 2 ? 6 : 4;
};

// shared memory: the warps' rings, the inputs, and the squares' sums of all columns;
// the totals lie over rings and inputs at the end
struct Layout {
  int x, sq, total;                // bytes
};
template <int NB, int MT, int G, bool CENTER>
__host__ __device__ inline Layout layout(int warps, int cols, int chunk, int units, bool norm) {
  using R = Ring<MT, G, CENTER>;
  Layout l;
  l.x = warps * R::kSlots * R::kSlot;
  l.sq = l.x + (chunk + kPad) * 2 * cols;
  l.total = l.sq + (norm ? (units * R::U + kSquares - 1) / kSquares * kQ4Rows * 4 : 0);
  return l;
}

__device__ __forceinline__ void copy16(char* to, const char* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                   (unsigned)__cvta_generic_to_shared(to)),
               "l"(from)
               : "memory");
}

template <typename T, int NB, int MT, int G, bool CENTER>
__global__ void __launch_bounds__(256, 2) rows_q4_kernel(const RowsQ4Params p) {
  using R = Ring<MT, G, CENTER>;
  constexpr int U = R::U, BU = R::BU;
  extern __shared__ __align__(16) char smem[];
  __shared__ float s_rstd[kQ4Rows];
  const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int mw = warp % p.mw, kw = warp / p.mw;
  const int units = (p.d_in + U - 1) / U, per = (units - kw + p.kw - 1) / p.kw;   // of this warp
  const int parts = sizeof(T) == 4 || p.norm_w != nullptr ? 3 : 1, cols = parts * p.rows;
  const int chunk_units = p.chunk / U, per_chunk = chunk_units / p.kw;
  const Layout lay = layout<NB, MT, G, CENTER>(p.mw * p.kw, cols, p.chunk, units,
                                               p.norm_w != nullptr);
  char* ring = smem + warp * R::kSlots * R::kSlot;
  char* rows = smem + lay.x;
  float* sq = reinterpret_cast<float*>(smem + lay.sq);
  const int tiles = (p.d_out + 15) / 16, tile0 = (blockIdx.x * p.mw + mw) * MT;
  pdl_launch_dependents();

  // This warp's units kw, kw + p.kw, ..: the next one to copy.  A tile past the last is
  // the last once more; its results are not stored.
  const char* codes[MT];
  const char* scales[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const size_t at = (size_t)min(tile0 + m, tiles - 1) * units + kw;
    codes[m] = reinterpret_cast<const char*>(p.codes) + at * (BU * 512) + lane * 16;
    scales[m] = static_cast<const char*>(p.scales) + at * R::kScale + lane * 16;
  }
  int put = 0, slot_in = 0;
  auto copy = [&] {
    if (put < per) {
      char* to = ring + slot_in * R::kSlot + lane * 16;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int b = 0; b < BU; ++b) copy16(to + (m * BU + b) * 512, codes[m] + b * 512);
        if (lane < R::kScale / 16) copy16(to + MT * BU * 512 + m * R::kScale, scales[m]);
        codes[m] += (size_t)p.kw * (BU * 512);
        scales[m] += (size_t)p.kw * R::kScale;
      }
      ++put;
      slot_in = slot_in + 1 == R::kSlots ? 0 : slot_in + 1;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < R::kSlots - 1; ++i) copy();
  pdl_wait();
  // the bias and residual of this thread's first output
  const int outs = 16 * MT * p.mw, o_r = threadIdx.x / outs, o_at = blockIdx.x * outs + threadIdx.x % outs;
  float add_bias = 0.f, add_res = 0.f;
  if (o_r < p.rows && o_at < p.d_out) {
    if (p.bias != nullptr) add_bias = p.bias[o_at];
    if (p.residual != nullptr)
      add_res = Elem<T>::get(static_cast<const T*>(p.residual)[(size_t)o_r * p.ld_r + o_at]);
  }
  // the lane's operands of block 0; lanes of columns that are not in use read the last
  // one's, and their results are not used
  const char* mine[NB];
#pragma unroll
  for (int c = 0; c < NB; ++c)
    mine[c] = rows + min(c * 8 + (lane >> 2), cols - 1) * (p.chunk + kPad) * 2 + (lane & 3) * 16;
  float tot[MT][NB][4] = {};
  int slot = 0;
  for (int i0 = 0; i0 * p.kw < units; i0 += per_chunk) {   // chunks of the columns
    const int u0 = i0 * p.kw;
    __syncthreads();
    stage<T>(p, u0 * U, min(chunk_units, units - u0) * U, rows, sq, parts);
    __syncthreads();
    const int end = min(per, i0 + per_chunk);
    for (int i = i0; i < end; ++i) {
      copy();
      asm volatile("cp.async.wait_group %0;" ::"n"(R::kSlots - 1) : "memory");
      __syncwarp();
      const char* from = ring + slot * R::kSlot;
      slot = slot + 1 == R::kSlots ? 0 : slot + 1;
      const int u = (i - i0) * p.kw + kw;            // in the chunk
      float acc[MT][NB][4], sum[NB][4];              // sum: of the inputs, in every row
#pragma unroll
      for (int b = 0; b < BU; ++b) {
        uint4 w[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m)
          w[m] = *reinterpret_cast<const uint4*>(from + (m * BU + b) * 512 + lane * 16);
#pragma unroll
        for (int jp = 0; jp < 2; ++jp) {             // two instructions' worth of columns
          const bool first = G < 64 || (b == 0 && jp == 0), last = G < 64 || (b == BU - 1 && jp == 1);
          uint4 f[NB];
#pragma unroll
          for (int c = 0; c < NB; ++c)
            f[c] = *reinterpret_cast<const uint4*>(mine[c] + (u * BU + b) * 128 + jp * 64);
          if (CENTER) {
            constexpr unsigned kOnes = 0x3f803f80u;
            const unsigned one[4] = {kOnes, kOnes, kOnes, kOnes};
#pragma unroll
            for (int c = 0; c < NB; ++c) {
              if (first) sum[c][0] = sum[c][1] = sum[c][2] = sum[c][3] = 0.f;
              mma16816(sum[c], one, f[c].x, f[c].y);
              mma16816(sum[c], one, f[c].z, f[c].w);
            }
          }
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            if (first)
#pragma unroll
              for (int c = 0; c < NB; ++c)
                acc[m][c][0] = acc[m][c][1] = acc[m][c][2] = acc[m][c][3] = 0.f;
            unsigned a[4];
            unpack(jp ? w[m].z : w[m].x, a);
#pragma unroll
            for (int c = 0; c < NB; ++c) mma16816(acc[m][c], a, f[c].x, f[c].y);
            unpack(jp ? w[m].w : w[m].y, a);
#pragma unroll
            for (int c = 0; c < NB; ++c) mma16816(acc[m][c], a, f[c].z, f[c].w);
            if (last) {
              const int g = G < 64 ? jp : 0;
              const char* sp = from + MT * BU * 512 + m * R::kScale;
              float s0, s1, c0 = 0.f, c1 = 0.f;      // of outputs lane / 4 and lane / 4 + 8
              if (CENTER) {
                const uint2 s2 = reinterpret_cast<const uint2*>(sp)[g * 8 + (lane >> 2)];
                s0 = __uint_as_float(s2.x << 16);
                c0 = __uint_as_float(s2.x & 0xffff0000u);
                s1 = __uint_as_float(s2.y << 16);
                c1 = __uint_as_float(s2.y & 0xffff0000u);
              } else {
                const unsigned s2 = reinterpret_cast<const unsigned*>(sp)[g * 8 + (lane >> 2)];
                s0 = __uint_as_float(s2 << 16);
                s1 = __uint_as_float(s2 & 0xffff0000u);
              }
#pragma unroll
              for (int c = 0; c < NB; ++c) {
                tot[m][c][0] = fmaf(s0, acc[m][c][0], tot[m][c][0]);
                tot[m][c][1] = fmaf(s0, acc[m][c][1], tot[m][c][1]);
                tot[m][c][2] = fmaf(s1, acc[m][c][2], tot[m][c][2]);
                tot[m][c][3] = fmaf(s1, acc[m][c][3], tot[m][c][3]);
                if (CENTER) {
                  tot[m][c][0] = fmaf(c0, sum[c][0], tot[m][c][0]);
                  tot[m][c][1] = fmaf(c0, sum[c][1], tot[m][c][1]);
                  tot[m][c][2] = fmaf(c1, sum[c][0], tot[m][c][2]);
                  tot[m][c][3] = fmaf(c1, sum[c][1], tot[m][c][3]);
                }
              }
            }
          }
        }
      }
      __syncwarp();                                  // before the slot is copied to again
    }
  }

  // the rows' 1 / sqrt(mean(x^2) + eps): 128 columns at a time, strided over a warp's lanes
  if (p.norm_w != nullptr)
    for (int r = warp; r < p.rows; r += blockDim.x >> 5) {
      float v = 0.f;
      for (int u = lane; u * kSquares < p.d_in; u += 32) v += sq[u * kQ4Rows + r];
      v = warp_total(v, 32);
      if (lane == 0) s_rstd[r] = rsqrtf(v / (float)p.d_in + p.eps);
    }
  __syncthreads();
  // totals of every warp: (kw, outputs of the CTA, columns)
  float* red = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int c = 0; c < NB; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int o = (mw * MT + m) * 16 + (lane >> 2) + (i >> 1) * 8;
        red[((size_t)kw * outs + o) * (8 * NB + 1) + c * 8 + 2 * (lane & 3) + (i & 1)] =
            tot[m][c][i];
      }
  __syncthreads();
  for (int i = threadIdx.x; i < outs * p.rows; i += blockDim.x) {
    const int r = i / outs, o = i - r * outs, out = blockIdx.x * outs + o;
    if (out >= p.d_out) continue;
    float v = 0.f;
    for (int s = parts - 1; s >= 0; --s)             // the smallest part first
      for (int k = 0; k < p.kw; ++k)
        v += red[((size_t)k * outs + o) * (8 * NB + 1) + s * p.rows + r];
    if (p.norm_w != nullptr) v *= s_rstd[r];
    if (i != threadIdx.x) {
      add_bias = p.bias != nullptr ? p.bias[out] : 0.f;
      add_res = p.residual != nullptr
                    ? Elem<T>::get(static_cast<const T*>(p.residual)[(size_t)r * p.ld_r + out])
                    : 0.f;
    }
    v = add_res + (v + add_bias);
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
  constexpr int U = G > 64 ? G : 64;
  constexpr int kSmem = 112 << 10;                   // two CTAs per SM
  const int units = (p.d_in + U - 1) / U;
  const bool norm = p.norm_w != nullptr;
  const int cols = p.rows * (sizeof(T) == 4 || norm ? 3 : 1);
  // As many columns at a time as fit, a whole number of units of every warp, of fewer
  // warps where one unit of each does not fit (at one warp along the columns it does:
  // the rings' 68 KB, 128 columns' 7 KB and 16 KB of squares' sums at d_in = kQ4MaxIn).
  // The norm's squares are summed by 128 columns, so every chunk but the last is whole
  // ones of these.
  auto bytes = [&](int chunk) {
    return layout<NB, MT, G, CENTER>(p.mw * p.kw, cols, chunk, units, norm).total;
  };
  auto step_of = [&](int kw) {
    const int one = kw * U;
    return norm && one % kSquares != 0 && units > kw ? 2 * one : one;
  };
  while (p.kw > 1 && bytes(step_of(p.kw)) > kSmem) --p.kw;
  const int step = step_of(p.kw);
  int chunk = (units * U + step - 1) / step * step;
  while (chunk > step && bytes(chunk) > kSmem) chunk -= step;
  p.chunk = chunk;
  const int red = p.kw * 16 * MT * p.mw * (8 * NB + 1) * 4;
  const int smem = bytes(chunk) > red ? bytes(chunk) : red;
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
  // Warps along the columns while tiles are few, along the outputs where there are more
  // than one wave of CTAs: fewer copies of the inputs are staged (65536 outputs, 3 rows
  // of 8192 bf16: 256 CTAs 79 us, 512 90, 1024 101; 3000 outputs, 8 rows of 6000: 188 CTAs
  // 35, 94 32, 47 39).  As many as fill the wave: 40000 outputs, 8 rows of 8192 fp32 5
  // warps 163, 8 warps in fewer CTAs 187; 50000, 8 rows of 4096 bf16 6 warps 36, 8 45.
  int mt = 1, mw = 1;
  if (tiles > 2LL * p.sms) mt = 2;
  const long long wave = 2LL * p.sms * mt;
  if (tiles > wave) mw = tiles > 8 * wave ? 8 : (int)((tiles + wave - 1) / wave);
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
