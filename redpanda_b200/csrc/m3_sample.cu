// Drawing one token per row from logits, by the inverse of the cumulative
// distribution at a given uniform number.
//
//   w_i = exp((x_i - max) / T); candidates: x_i neither -infinity nor NaN
//   order: x descending, then index ascending
//   top-k: the first k;  top-p: of those, the shortest prefix whose weight
//   reaches p times theirs (at least one);  min-p: w_i >= min_p
//   token: the smallest index whose cumulative weight, over the kept tokens in
//   index order, exceeds u times their total
// T <= 0 takes the first token of the order; a row without candidates gives -1.
//
// Whether a token is kept and which one is drawn hang on comparisons of sums,
// so the sums are exact: a weight is evaluated in double precision and rounded
// once to a 64-bit integer in units of 2^-shift (sums of V weights stay below
// 2^63).  Integer addition is associative, so shared-memory atomics and any
// thread order give the same sums, and results do not depend on scheduling.
//
// One CTA per row, which stays in shared memory when it fits (read once from
// HBM; longer rows are read again from L2).  The bound is the double-precision
// exponential of every token whose weight counts, so as few as possible are
// evaluated:
//  - temperature 0 and k = 1 need the maximum only;
//  - up to kList tokens in play (few candidates, or a top-k whose histogram of
//    1024 bins over (max - x) / T, 32 per unit, ends early): they are gathered,
//    one per thread, ranked by comparing all pairs, and everything else happens
//    among them;
//  - a top-p or min-p without a top-k: the total is summed in fp32 with a known
//    error, the kLong first tokens of the order (no more than min-p leaves) are
//    gathered with exact weights, and the top-p border is looked for among them.
//    A border nearer to p times the total than the error allows, or one behind
//    the gathered tokens, is left to the next way;
//  - otherwise a top-k or top-p prefix ends in one bin of that histogram (of
//    counts, or of exact weights); the bin's members are gathered and ranked.  A
//    bin with more than kList members (ties) is cut down by 8-bit digits of the
//    ordered key.
// Measured for 4096 rows of 8192 bf16 logits, top-p and min-p of their own per
// row, half of them with k = 1: 589 us with every way by digits and the
// library's exponential, 164 us without the gathered lists, 105 us with the
// row cached as floats, 91 us now (the row's bytes alone: 10 us; it is bound by
// instructions, about 70 per token on average).  Shorter lists (kLong 512) or
// fewer bins (512) free room for another CTA but leave more rows to the next way:
// 100 and 96 us.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include "m3_api_util.h"
#include "m3_math.cuh"
#include "m3_ops.h"
#include "m3_vec.cuh"

namespace m3 {
namespace {

typedef unsigned long long u64;
constexpr int kBins = 1024;
constexpr float kBinsPerUnit = 32.f;
constexpr int kCacheMax = 32768;   // logits of a row kept in shared memory
constexpr int kList = 256;         // tokens ranked by comparing all pairs
constexpr int kLong = 1024;        // tokens gathered around a top-p or min-p border
// Bound on the relative error of the fp32 total of a row's weights, in steps of
// e = 2^-24 and to first order.
//  - The exponent y = (x - max) c, c = log2(e) / T, passes 4.3 roundings (the
//    difference, 1 / T, log2(e) itself, two products), so a weight 2^y is off by
//    ln 2 * 4.3 |y| e < 3 |y| e.  Over the weights' own distribution the mean of |y|
//    is its entropy less log2 of the total (which is 1 at least): at most log2 V
//    <= 18, so 54 e of the total.
//  - ex2.approx: 4 e.  The exact weights' own rounding to integers: below e.
//  - The additions that a weight passes: its thread's (V / NT, 5 more where four
//    neighbours go together), 5 shuffles, NT / 32 warps.
template <int NT>
__device__ __forceinline__ double sum_error(int V) {
  return (54 + 4 + 1 + V / NT + 5 + 5 + NT / 32) * 0x1p-24;
}

// A key whose unsigned order is x descending.
__device__ __forceinline__ unsigned desc_key(float x) {
  const unsigned b = __float_as_uint(x + 0.f);   // -0 and 0 are ties
  return (b & 0x80000000u) ? b : ~(b | 0x80000000u);
}

struct Shared {
  unsigned count[kBins];           // counts, or the low words of the weights
  unsigned high[kBins];            // the high words
  u64 wsum[33];
  double pow2[32];                 // 2^(j/32)
  u64 lw[kLong], sw[kList];
  float lx[kList];
  int mi[kList];
  int mn;
  int li[kLong];
  float fsum[32];
  int ln;
  u64 found_base;
  int found;
  int imax;
  float wm[32];
  int wi[32];
};

// Adds to a 64-bit counter kept as two words.
__device__ __forceinline__ void add64(Shared& sh, int i, u64 w) {
  const unsigned lo = (unsigned)w, old = atomicAdd(&sh.count[i], lo);
  const unsigned hi = (unsigned)(w >> 32) + (old + lo < old ? 1u : 0u);
  if (hi) atomicAdd(&sh.high[i], hi);
}
__device__ __forceinline__ u64 get_bin(const Shared& sh, bool mass, int i) {
  return mass ? ((u64)sh.high[i] << 32 | sh.count[i]) : (u64)sh.count[i];
}

// Exclusive prefix of v over the CTA's threads; *total gets the sum.
template <int NT>
__device__ u64 block_prefix(u64 v, u64* wsum, u64* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 s = v;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const u64 o = __shfl_up_sync(0xffffffffu, s, m);
    if (lane >= m) s += o;
  }
  if (lane == 31) wsum[warp] = s;
  __syncthreads();
  // every warp scans the warps' sums
  u64 t = lane < NT / 32 ? wsum[lane] : 0;
#pragma unroll
  for (int m = 1; m < NT / 32; m <<= 1) {
    const u64 o = __shfl_up_sync(0xffffffffu, t, m);
    if (lane >= m) t += o;
  }
  const u64 base = __shfl_sync(0xffffffffu, t, warp > 0 ? warp - 1 : 0);
  *total = __shfl_sync(0xffffffffu, t, NT / 32 - 1);
  __syncthreads();
  return (warp > 0 ? base : 0) + s - v;
}

// The bin where the running sum of the histogram (counts, or masses) first
// reaches thr, with the sum before it; nbins a multiple of NT or below it.
template <int NT>
__device__ void find_bin(Shared& sh, bool mass, int nbins, u64 thr) {
  const int per = nbins / NT > 0 ? nbins / NT : 1;
  const int i0 = threadIdx.x * per;
  u64 s = 0;
  if (i0 < nbins)
    for (int i = 0; i < per; ++i) s += get_bin(sh, mass, i0 + i);
  u64 total;
  u64 base = block_prefix<NT>(s, sh.wsum, &total);
  if (i0 < nbins && base < thr && base + s >= thr) {
    for (int i = 0; i < per; ++i) {
      const u64 v = get_bin(sh, mass, i0 + i);
      if (base + v >= thr) {
        sh.found = i0 + i;
        sh.found_base = base;
        break;
      }
      base += v;
    }
  }
  __syncthreads();
}

// A prefix of the order: keys below `key`, and of that key the indices up to
// `last`.
struct Cut {
  unsigned key = 0xffffffffu;
  int last = 0x7fffffff;
  __device__ __forceinline__ bool has(unsigned k, int i) const {
    return k < key || (k == key && i <= last);
  }
};

// The row: cached in its own type, where two bytes a token hold two more CTAs per
// SM than four, or the logits themselves (NaN as -infinity).
template <typename T, bool CACHE>
struct RowReader {
  const T* g;
  const T* s;
  __device__ __forceinline__ float at(int i) const {
    if (CACHE) return Elem<T>::get(s[i]);
    const float v = Elem<T>::get(g[i]);
    return v > -CUDART_INF_F ? v : -CUDART_INF_F;
  }
};

__device__ __forceinline__ void cache_four(float* p, float4 f) {
  *reinterpret_cast<float4*>(p) = f;
}
__device__ __forceinline__ void cache_four(__nv_bfloat16* p, float4 f) {
  __nv_bfloat162 v[2] = {__floats2bfloat162_rn(f.x, f.y), __floats2bfloat162_rn(f.z, f.w)};
  *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(v);
}

template <typename T, int NT, bool CACHE>
__global__ void __launch_bounds__(NT) sample_kernel(const SampleParams p) {
  extern __shared__ __align__(16) unsigned char raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw);
  T* cache = reinterpret_cast<T*>(raw + (sizeof(Shared) + 15) / 16 * 16);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const size_t row = blockIdx.x;
  const int V = p.V;
  const T* g = static_cast<const T*>(p.logits) + row * p.ld;
  const RowReader<T, CACHE> x{g, cache};

  // ---- maximum and candidates
  float m = -CUDART_INF_F;
  unsigned cand = 0;
  auto look = [&](float v) -> float {
    v = fmaxf(v, -CUDART_INF_F);   // NaN as -infinity
    m = fmaxf(m, v);
    cand += v > -CUDART_INF_F;
    return v;
  };
  constexpr int VW = 16 / (int)sizeof(T);
  const int head = p.vec ? V / VW * VW : 0;
  constexpr int UNR = 4;      // loads in flight per thread
  for (int i0 = tid * VW; i0 < head; i0 += NT * VW * UNR) {
    Pack<T, VW> v[UNR];
#pragma unroll
    for (int k = 0; k < UNR; ++k)
      if (i0 + k * NT * VW < head) v[k] = ld_pack<T, VW>(g + i0 + k * NT * VW);
#pragma unroll
    for (int k = 0; k < UNR; ++k) {
      const int i = i0 + k * NT * VW;
      if (i < head) {
#pragma unroll
        for (int j = 0; j < VW; j += 4) {
          const float4 f = make_float4(look(v[k].get(j)), look(v[k].get(j + 1)),
                                       look(v[k].get(j + 2)), look(v[k].get(j + 3)));
          if (CACHE) cache_four(cache + i + j, f);
        }
      }
    }
  }
  for (int i = head + tid; i < V; i += NT) {
    const float v = look(Elem<T>::get(g[i]));
    if (CACHE) cache[i] = Elem<T>::put(v);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    cand += __shfl_xor_sync(0xffffffffu, cand, o);
  }
  if (tid == 0) { sh.ln = 0; sh.imax = 0x7fffffff; }
  if (lane == 0) { sh.wm[warp] = m; sh.wi[warp] = (int)cand; }
  __syncthreads();
  float top = sh.wm[0];
  int ncand = sh.wi[0];
#pragma unroll
  for (int w = 1; w < NT / 32; ++w) {
    top = fmaxf(top, sh.wm[w]);
    ncand += sh.wi[w];
  }
  // every token, four at a time from the cache
  auto for_each = [&](auto&& f) {
    if (CACHE) {
      const int whole = V & ~3;
      for (int i = 4 * tid; i < whole; i += 4 * NT) {
        const Pack<T, 4> v = ld_pack<T, 4>(cache + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) f(i + j, v.get(j));
      }
      if (whole + tid < V) f(whole + tid, x.at(whole + tid));
    } else {
#pragma unroll 4
      for (int i = tid; i < V; i += NT) f(i, x.at(i));
    }
  };
  const float temp = p.temperature ? p.temperature[row] : p.temperature0;
  const int k = p.top_k ? p.top_k[row] : p.top_k0;
  if (ncand == 0 || !(temp > 0.f) || k == 1) {   // the first token of the order
    for_each([&](int i, float v) {
      if (v == top && ncand) atomicMin(&sh.imax, i);
    });
    __syncthreads();
    if (tid == 0) p.out[row] = ncand ? sh.imax : -1;
    return;
  }
  if (tid < 32) sh.pow2[tid] = exp2((double)tid / 32);
  __syncthreads();   // the draw without any cut evaluates weights at once
  // NaN and negative as 0, the first token: each of the ways below compares tp in
  // its own direction
  const float tp = fmaxf(p.top_p ? p.top_p[row] : p.top_p0, 0.f);
  const double mp = fmin((double)(p.min_p ? p.min_p[row] : p.min_p0), 1.0);
  const double dtop = (double)top, unit = exp2((double)p.shift);
  const double scale = CUDART_L2E / (double)temp;   // to powers of 2
  const float inv_t = 1.f / temp;

  // 2^y for y <= 0 by the table of 2^(j/32) and the exponential series of the
  // rest, |r| <= ln 2 / 64 (P. T. P. Tang, "Table-driven implementation of the
  // exponential function", ACM TOMS 15, 1989): 14 double-precision operations.
  auto weight = [&](float v) -> double {
    if (v == top) return 1.0;
    const double y = ((double)v - dtop) * scale;
    if (!(y > -1000.0)) return 0.0;
    constexpr double kShifter = 6755399441055744.0;   // 1.5 * 2^52
    const double t = fma(y, 32.0, kShifter);
    const int k32 = __double2loint(t);
    const double r = fma(t - kShifter, -1.0 / 32, y) * CUDART_LN2;
    double e = 1.0 / 720;
    e = fma(e, r, 1.0 / 120);
    e = fma(e, r, 1.0 / 24);
    e = fma(e, r, 1.0 / 6);
    e = fma(e, r, 0.5);
    e = fma(e, r, 1.0);
    e = fma(e, r, 1.0) * sh.pow2[k32 & 31];
    return __hiloint2double(__double2hiint(e) + ((k32 >> 5) << 20), __double2loint(e));
  };
  // shift <= 50: the integer stands in the low bits of the shifted sum
  auto in_units = [&](double w) -> u64 {
    return (u64)__double_as_longlong(fma(w, unit, 4503599627370496.0)) & 0xfffffffffffffull;
  };
  auto units = [&](float v) -> u64 { return in_units(weight(v)); };
  // a bin of the order: monotone in v, equal values share it
  auto bin_of = [&](float v) -> int {
    const float d = (top - v) * inv_t * kBinsPerUnit;
    return v == top ? 0 : d < (float)(kBins - 1) ? (int)d : kBins - 1;
  };

  auto clear = [&](int n, bool mass) {
    __syncthreads();
    for (int i = tid; i < n; i += NT) {
      sh.count[i] = 0;
      if (mass) sh.high[i] = 0;
    }
    __syncthreads();
  };
  // The number of the target: the smallest cumulative weight to reach.
  auto target = [&](u64 total) -> u64 {
    const double at = (double)p.u[row] * (double)total;
    const u64 thr = at > 0.0 ? (at < (double)total ? (u64)at + 1 : total) : 1;
    return thr > total ? total : thr;
  };

  // ---- few tokens in play: among those that f names (at most kList)
  auto finish = [&](auto&& f) {
    for_each([&](int i, float v) {
      if (v > -CUDART_INF_F && f(v)) {
        const int at = atomicAdd(&sh.ln, 1);
        if (at < kList) { sh.lx[at] = v; sh.li[at] = i; }
      }
    });
    __syncthreads();
    const int n = sh.ln;
    float mx = 0.f;
    int mi = 0, rank = 0;
    double w = 0.0;
    if (tid < n) {
      mx = sh.lx[tid];
      mi = sh.li[tid];
      for (int j = 0; j < n; ++j)
        rank += sh.lx[j] > mx || (sh.lx[j] == mx && sh.li[j] < mi);
      w = weight(mx);
      sh.sw[rank] = (k <= 0 || rank < k) ? in_units(w) : 0;
    }
    __syncthreads();
    // thread r looks at the token of rank r: is it in the top-p prefix?
    u64 total;
    const u64 own = tid < n ? sh.sw[tid] : 0;
    const u64 before = block_prefix<NT>(own, sh.wsum, &total);
    if (tid < n && !(tid == 0 || tp >= 1.f || (double)before < (double)tp * (double)total))
      sh.sw[tid] = 0;
    __syncthreads();
    u64 mine = 0;
    if (tid < n) {
      mine = w >= mp ? sh.sw[rank] : 0;
      sh.lw[tid] = mine;
    }
    block_prefix<NT>(mine, sh.wsum, &total);   // its barriers show lw too
    const u64 thr = target(total);
    if (mine) {
      u64 cum = 0;
      for (int j = 0; j < n; ++j) cum += sh.li[j] <= mi ? sh.lw[j] : 0;
      if (cum >= thr && cum - mine < thr) p.out[row] = mi;
    }
  };
  if (ncand <= kList) {
    finish([](float) { return true; });
    return;
  }

  Cut cut;
  // The cut of the shortest prefix (of what `cut` keeps) whose measure reaches
  // thr: counts, or weights.  It ends in bin `bin`, with `base` before the bin.
  auto select = [&](bool mass, u64 thr, int bin, u64 base) {
    if (tid == 0) sh.ln = 0;
    __syncthreads();
    for_each([&](int i, float v) {
      if (v > -CUDART_INF_F && bin_of(v) == bin && cut.has(desc_key(v), i)) {
        const int at = atomicAdd(&sh.ln, 1);
        if (at < kList) { sh.lx[at] = v; sh.li[at] = i; }
      }
    });
    __syncthreads();
    const int n = sh.ln;
    Cut c;
    if (n <= kList) {   // rank the bin's members
      if (tid < n) sh.lw[tid] = mass ? units(sh.lx[tid]) : 1;
      __syncthreads();
      if (tid < n) {
        const float mx = sh.lx[tid];
        const int mi = sh.li[tid];
        u64 upto = base;   // this member included
        for (int j = 0; j < n; ++j)
          upto += (sh.lx[j] > mx || (sh.lx[j] == mx && sh.li[j] <= mi)) ? sh.lw[j] : 0;
        if (upto >= thr && upto - sh.lw[tid] < thr) sh.found = tid;
      }
      __syncthreads();
      const int at = min(sh.found, kList - 1);
      c.key = desc_key(sh.lx[at]);
      c.last = sh.li[at];
      __syncthreads();
      cut = c;
      return;
    }
    unsigned prefix = 0;
    for (int level = 3; level >= 0; --level) {
      const int sft = level * 8;
      clear(256, true);
      for (int i = tid; i < V; i += NT) {
        const float v = x.at(i);
        if (!(v > -CUDART_INF_F) || bin_of(v) != bin) continue;
        const unsigned key = desc_key(v);
        if (!cut.has(key, i) || (level < 3 && (key >> (sft + 8)) != (prefix >> (sft + 8))))
          continue;
        if (mass) add64(sh, key >> sft & 255, units(v));
        else atomicAdd(&sh.count[key >> sft & 255], 1u);
      }
      __syncthreads();
      find_bin<NT>(sh, mass, 256, thr - base);
      prefix |= (unsigned)sh.found << sft;
      base += sh.found_base;
    }
    // one value is left: how many of its ties to keep
    c.key = prefix;
    u64 need = thr - base;
    if (mass) {
      const unsigned b = prefix & 0x80000000u ? prefix : ~prefix & 0x7fffffffu;
      const u64 each = units(__uint_as_float(b));
      need = (need + each - 1) / each;
    }
    // the need-th tie by index: warps own runs of indices
    const int seg = (V + NT / 32 - 1) / (NT / 32), s0 = warp * seg, s1 = min(s0 + seg, V);
    auto tie = [&](int i) {
      return i < s1 && x.at(i) > -CUDART_INF_F && desc_key(x.at(i)) == prefix &&
             cut.has(prefix, i);
    };
    unsigned mine = 0;
    for (int i = s0 + lane; i - lane < s1; i += 32)
      mine += __popc(__ballot_sync(0xffffffffu, tie(i)));
    __syncthreads();
    if (lane == 0) sh.wsum[warp] = mine;
    if (tid == 0) sh.found = cut.key == prefix ? cut.last : 0x7fffffff;   // all of them
    __syncthreads();
    u64 before = 0;
    for (int w = 0; w < warp; ++w) before += sh.wsum[w];
    if (before < need && before + mine >= need) {
      u64 left = need - before;
      for (int i = s0 + lane; i - lane < s1; i += 32) {
        const bool t = tie(i);
        const unsigned bits = __ballot_sync(0xffffffffu, t);
        const unsigned cnt = __popc(bits);
        if (cnt >= left) {
          if (t && __popc(bits & ((2u << lane) - 1)) == left) sh.found = i;
          break;
        }
        left -= cnt;
      }
    }
    __syncthreads();
    c.last = sh.found;
    __syncthreads();
    cut = c;
  };

  // ---- top-p and min-p among the first tokens of the order; false: not decided
  auto among_first = [&]() -> bool {
    if (top == CUDART_INF_F) return false;
    clear(kBins, false);
    // bins of this way, monotone in v like bin_of: from the weight's own exponent
    const float c2 = inv_t * 1.44269504f;
    constexpr float kBinsPerPower = -kBinsPerUnit * 0.693147181f;
    auto bin2 = [&](float v) -> int {
      return (int)fminf((v - top) * c2 * kBinsPerPower, (float)(kBins - 1));
    };
    float sum = 0.f;
    for_each([&](int, float v) {
      const float y = (v - top) * c2;
      sum += ex2_approx(y);
      if (v > -CUDART_INF_F)
        atomicAdd(&sh.count[(int)fminf(y * kBinsPerPower, (float)(kBins - 1))], 1u);
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sh.fsum[warp] = sum;
    __syncthreads();
    float all = 0.f;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) all += sh.fsum[w];
    // the bins in play: kLong tokens at most, none that min-p drops
    int bins = kBins;
    if (mp > 0.0) {
      const float d = -logf((float)mp) * kBinsPerUnit + 2.f;   // in bins, one to spare
      if (d < (float)kBins) bins = (int)d;
    }
    if (tid == 0) { sh.found = -1; sh.ln = 0; }
    __syncthreads();
    {
      const int per = kBins / NT, i0 = tid * per;
      u64 mine = 0, total;
      for (int i = 0; i < per; ++i) mine += sh.count[i0 + i];
      u64 run = block_prefix<NT>(mine, sh.wsum, &total);
      for (int i = 0; i < per; ++i) {
        run += sh.count[i0 + i];
        if (run <= (u64)kLong) atomicMax(&sh.found, i0 + i);
      }
    }
    __syncthreads();
    const int last = min(sh.found, bins - 1);
    const bool whole = last == bins - 1;   // min-p's tokens, or all, are gathered
    if (last < 0 || (tp >= 1.f && !whole)) return false;
    // (the last bin takes every weight below e^-32: its test is not this one)
    if (last == kBins - 1) return false;
    for_each([&](int i, float v) {
      if (v > -CUDART_INF_F && (v - top) * c2 * kBinsPerPower < (float)(last + 1)) {
        const int at = atomicAdd(&sh.ln, 1);
        if (at < kLong) sh.li[at] = i;
      }
    });
    __syncthreads();
    const int n = min(sh.ln, kLong);
    u64 mine = 0, got;
    for (int j = tid; j < n; j += NT) mine += sh.lw[j] = units(x.at(sh.li[j]));
    block_prefix<NT>(mine, sh.wsum, &got);
    // Gathered tokens that f names, one per thread (lx, mi, sw); their number, 0 when
    // they are too many.
    auto members = [&](auto&& f) -> int {
      __syncthreads();
      if (tid == 0) sh.mn = 0;
      __syncthreads();
      for (int j = tid; j < n; j += NT) {
        const int i = sh.li[j];
        if (sh.lw[j] && f(i)) {
          const int at = atomicAdd(&sh.mn, 1);
          if (at < kList) {
            sh.lx[at] = x.at(i);
            sh.mi[at] = i;
            sh.sw[at] = sh.lw[j];
          }
        }
      }
      __syncthreads();
      return sh.mn <= kList ? sh.mn : 0;
    };
    Cut c;
    if (tp < 1.f) {
      const double want = (double)tp * (double)all * unit, slack = sum_error<NT>(V) * want + 1.0;
      if ((double)got < want + slack) {
        if (!whole || (double)got > want - slack) return false;
        // top-p's border is behind min-p's: everything gathered stays
      } else {
        // the first token at which the running weight reaches `want`
        clear(kBins, true);
        for (int j = tid; j < n; j += NT)
          if (sh.lw[j]) add64(sh, bin2(x.at(sh.li[j])), sh.lw[j]);
        __syncthreads();
        const u64 thr = want >= 1.0 ? (u64)ceil(want) : 1ull;
        find_bin<NT>(sh, true, kBins, thr);
        const int bin = sh.found;
        const u64 base = sh.found_base;
        const int m = members([&](int i) { return bin2(x.at(i)) == bin; });
        if (tid == 0) sh.found = -1;
        __syncthreads();
        if (tid < m) {
          const float v = sh.lx[tid];
          u64 before = base;
          for (int o = 0; o < m; ++o)
            before += (sh.lx[o] > v || (sh.lx[o] == v && sh.mi[o] < sh.mi[tid])) ? sh.sw[o] : 0;
          const u64 upto = before + sh.sw[tid];
          // the order's first token always stays
          if (upto >= thr && before < thr && (double)upto > want + slack &&
              (before == 0 || (double)before < want - slack))
            sh.found = tid;
        }
        __syncthreads();
        if (sh.found < 0) return false;   // too near to call
        c.key = desc_key(sh.lx[sh.found]);
        c.last = sh.mi[sh.found];
      }
    }
    // draw: weights by runs of indices, then the run's members by index
    __syncthreads();
    const int shift_i = max(0, 32 - __clz(max(V - 1, 1)) - 8);   // 256 runs at most
    clear(kList, true);
    mine = 0;
    for (int j = tid; j < n; j += NT) {
      const int i = sh.li[j];
      const float v = x.at(i);
      u64 w = c.has(desc_key(v), i) ? sh.lw[j] : 0;
      if (w && mp > 0.0 && !(weight(v) >= mp)) w = 0;
      sh.lw[j] = w;
      mine += w;
      if (w) add64(sh, i >> shift_i, w);
    }
    u64 total;
    block_prefix<NT>(mine, sh.wsum, &total);
    const u64 thr = target(total);
    find_bin<NT>(sh, true, kList, thr);
    const int run = sh.found;
    const u64 base = sh.found_base;
    const int m = members([&](int i) { return i >> shift_i == run; });
    if (m == 0) return false;   // a run of more than kList tokens
    if (tid < m) {
      u64 cum = base;
      for (int o = 0; o < m; ++o) cum += sh.mi[o] <= sh.mi[tid] ? sh.sw[o] : 0;
      if (cum >= thr && cum - sh.sw[tid] < thr) p.out[row] = sh.mi[tid];
    }
    return true;
  };
  const bool limited = k > 0 && k < ncand;
  if (!limited && (tp < 1.f || mp > 0.0)) {
    if (among_first()) return;
    __syncthreads();
  }

  if (limited) {
    clear(kBins, false);
    for_each([&](int i, float v) {
      if (v > -CUDART_INF_F) atomicAdd(&sh.count[bin_of(v)], 1u);
    });
    __syncthreads();
    find_bin<NT>(sh, false, kBins, (u64)k);
    const int bin = sh.found;
    const u64 base = sh.found_base;
    if (base + sh.count[bin] <= kList) {   // the prefix's bins hold few tokens
      finish([&](float v) { return bin_of(v) <= bin; });
      return;
    }
    select(false, (u64)k, bin, base);
  }
  if (tp < 1.f) {
    clear(kBins, true);
    u64 mine = 0;
    for_each([&](int i, float v) {
      if (v > -CUDART_INF_F && cut.has(desc_key(v), i)) {
        const u64 w = units(v);
        mine += w;
        if (w) add64(sh, bin_of(v), w);
      }
    });
    u64 total;
    block_prefix<NT>(mine, sh.wsum, &total);
    const double want = ceil((double)tp * (double)total);
    const u64 thr = want >= 1.0 ? (u64)want : 1ull;   // p = 0: the first token
    find_bin<NT>(sh, true, kBins, thr);
    select(true, thr, sh.found, sh.found_base);
  }

  // ---- draw: warps own runs of indices
  const int seg = (V + NT / 32 - 1) / (NT / 32), s0 = warp * seg, s1 = min(s0 + seg, V);
  auto kept = [&](int i) -> u64 {
    if (i >= s1) return 0;
    const float v = x.at(i);
    if (!(v > -CUDART_INF_F) || !cut.has(desc_key(v), i)) return 0;
    const double w = weight(v);
    return w >= mp ? in_units(w) : 0;
  };
  u64 mine = 0;
  for (int i = s0 + lane; i - lane < s1; i += 32) mine += kept(i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  __syncthreads();
  if (lane == 0) sh.wsum[warp] = mine;
  __syncthreads();
  u64 before = 0, total = 0;
  for (int w = 0; w < NT / 32; ++w) {
    if (w < warp) before += sh.wsum[w];
    total += sh.wsum[w];
  }
  const u64 thr = target(total);
  if (before < thr && before + mine >= thr) {
    u64 run = before;
    for (int i = s0 + lane; i - lane < s1; i += 32) {
      u64 s = kept(i);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 a = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += a;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, run + s >= thr);
      if (hit) {
        if (lane == __ffs(hit) - 1) p.out[row] = i;
        break;
      }
      run += __shfl_sync(0xffffffffu, s, 31);
    }
  }
}

template <typename T, int NT, bool CACHE>
cudaError_t sample_typed(const SampleParams& p, cudaStream_t s) {
  constexpr auto* kern = sample_kernel<T, NT, CACHE>;
  const int smem = ((int)sizeof(Shared) + 15) / 16 * 16 + (CACHE ? (p.V + 3) / 4 * 4 * (int)sizeof(T) : 0);
  // the most that any row length takes: calls side by side set one value
  constexpr int most = ((int)sizeof(Shared) + 15) / 16 * 16 + (CACHE ? kCacheMax * (int)sizeof(T) : 0);
  const cudaError_t e = allow_smem<kern>(most);
  if (e != cudaSuccess) return e;
  kern<<<p.rows, NT, smem, s>>>(p);
  return cudaGetLastError();
}

template <typename T>
cudaError_t sample_rows(const SampleParams& p, cudaStream_t s) {
  if (p.V > kCacheMax) return sample_typed<T, 1024, false>(p, s);
  if (p.V > 4096 && p.rows <= 2 * p.sms) return sample_typed<T, 1024, true>(p, s);
  return sample_typed<T, 256, true>(p, s);
}

}  // namespace

cudaError_t launch_sample(const SampleParams& p0, cudaStream_t s) {
  SampleParams p = p0;
  p.vec = aligned(p.logits, 16) && p.ld % (16 / dsize(p.dtype)) == 0;
  return p.dtype == M3_BF16 ? sample_rows<__nv_bfloat16>(p, s) : sample_rows<float>(p, s);
}

}  // namespace m3
