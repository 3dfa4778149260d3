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

// rows of `ld` elements of size e that vectors of V elements may be read from
inline bool rows_ok(const void* p, long long ld, int e, int v) {
  return p == nullptr || (aligned(p, v * e < 16 ? v * e : 16) && ld % v == 0);
}

}  // namespace
}  // namespace m3
