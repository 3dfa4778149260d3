// Launch of the add-norm kernels: vector width and element types.
#pragma once

#include "m3_norm.cuh"
#include "m3_ops.h"

namespace m3 {
namespace {

// f<TX, TS, TY>() of the three element types
template <typename F>
cudaError_t with_types(int x, int s, int y, F&& f) {
  using B = __nv_bfloat16;
  auto third = [&](auto tx, auto ts) {
    return y == M3_BF16 ? f(tx, ts, B()) : f(tx, ts, float());
  };
  auto second = [&](auto tx) { return s == M3_BF16 ? third(tx, B()) : third(tx, float()); };
  return x == M3_BF16 ? second(B()) : second(float());
}

// Instantiation of a row length, as norm_dispatch, but with 16 elements per thread in
// rows past F's kFrom, 2048 (1024 in the 8-bit norm): these kernels hold two or three
// arrays, and a CTA of 512 threads with 8 elements each fills an SM by itself with too
// little in flight (16384 x 4096 bf16: forward 116 against 92 us, backward 137
// against 116).
template <int E, int MAXT, typename F>
cudaError_t add_size(int vec, int nt, F&& f) {
  if constexpr (std::decay_t<F>::kWide)
    if (vec == 8) return f.template operator()<8, E / 8, false, MAXT, 1>(nt);
  if (vec == 2) return f.template operator()<2, E / 2, false, MAXT, 1>(nt);
  return vec == 4 ? f.template operator()<4, E / 4, false, MAXT, 1>(nt)
                  : f.template operator()<1, E, false, MAXT, 1>(nt);
}
inline int add_elements(int d, int from) { return d <= from ? 8 : d <= 16384 ? 16 : 32; }
inline int add_threads(int d, int from) {
  const int e = add_elements(d, from);
  return (d + 32 * e - 1) / (32 * e) * 32;
}
template <typename F>
cudaError_t add_dispatch(int d, int vec, F&& f) {
  constexpr int from = std::decay_t<F>::kFrom;
  constexpr bool kWarpRows = std::decay_t<F>::kWarpRows;
  if (d <= 256) return norm_warp<8>(vec, f);
  if constexpr (kWarpRows) {
    if (d <= 512) return norm_warp<16>(vec, f);
    if (d <= 768) return norm_warp<24>(vec, f);
    if (d <= 1024) return norm_warp<32>(vec, f);
  }
  const int nt = add_threads(d, from);
  if constexpr (!kWarpRows || from > 1024)
    if (d <= from) return add_size<8, 768>(vec, nt, f);   // 80 registers
  if (d <= 8192) return add_size<16, 512>(vec, nt, f);
  return d <= 16384 ? add_size<16, 1024>(vec, nt, f) : add_size<32, 1024>(vec, nt, f);
}

// CTAs per SM of a forward kernel at `threads` per CTA, asked for once
template <auto* kern>
int add_resident(int threads) {
  static OncePerDevice known[33];
  return resident_ctas<kern>(known[threads / 32], threads, 0);
}

// rows of `ld` elements of size e that vectors of V elements may be read from.  Even rows
// that 4 do not fit take pairs: 8447 x 866 bf16 forward 13 us and backward 16 against 24
// and 27 by elements, 19438 x 2734 fp32 149 and 228 against 219 and 282, 3207 x 8186 bf16 in
// 8 bits 51 against 90.
inline bool rows_ok(const void* p, long long ld, int e, int v) {
  return p == nullptr || (aligned(p, v * e < 16 ? v * e : 16) && ld % v == 0);
}

}  // namespace
}  // namespace m3
