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
// One CTA per row.  A prefix of the order (top-k: count k; top-p: weight) ends
// in a bin of a 2048-bin histogram over (max - x) / T, 64 bins per unit: one
// pass over the row.  Only that bin's few members are looked at again, by
// 8-bit digits of the ordered key, down to one value and the number of its ties
// to keep.  The row stays in shared memory when it fits (read once from HBM);
// longer rows are read again from L2.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include "m3_api_util.h"
#include "m3_ops.h"
#include "m3_vec.cuh"

namespace m3 {
namespace {

typedef unsigned long long u64;
constexpr int kBins = 2048;
constexpr float kBinsPerUnit = 64.f;
constexpr int kCacheMax = 32768;   // floats of a row kept in shared memory

// A key whose unsigned order is x descending.
__device__ __forceinline__ unsigned desc_key(float x) {
  const unsigned b = __float_as_uint(x + 0.f);   // -0 and 0 are ties
  return (b & 0x80000000u) ? b : ~(b | 0x80000000u);
}

struct Shared {
  u64 mass[kBins];
  unsigned count[kBins];
  u64 wsum[33];
  u64 found_base;
  u64 found_mass;
  int found;
  float fmax;
  int imax;
  unsigned n;
};

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
  u64 base = 0, all = 0;
  for (int w = 0; w < NT / 32; ++w) {
    if (w < warp) base += wsum[w];
    all += wsum[w];
  }
  __syncthreads();
  *total = all;
  return base + s - v;
}

// The bin where the running sum of the histogram (counts, or masses) first
// reaches thr, with the sum before it; nbins a multiple of NT or below it.
template <int NT>
__device__ void find_bin(Shared& sh, bool mass, int nbins, u64 thr) {
  const int per = nbins / NT > 0 ? nbins / NT : 1;
  const int i0 = threadIdx.x * per;
  u64 s = 0;
  if (i0 < nbins)
    for (int i = 0; i < per; ++i) s += mass ? sh.mass[i0 + i] : (u64)sh.count[i0 + i];
  u64 total;
  u64 base = block_prefix<NT>(s, sh.wsum, &total);
  if (i0 < nbins && base < thr && base + s >= thr) {
    for (int i = 0; i < per; ++i) {
      const u64 v = mass ? sh.mass[i0 + i] : (u64)sh.count[i0 + i];
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

template <typename T, int NT, bool CACHE>
struct RowReader {
  const T* g;
  const float* s;
  __device__ __forceinline__ float at(int i) const {
    return CACHE ? s[i] : Elem<T>::get(g[i]);
  }
};

template <typename T, int NT, bool CACHE>
__global__ void __launch_bounds__(NT) sample_kernel(const SampleParams p) {
  extern __shared__ __align__(16) unsigned char raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw);
  float* cache = reinterpret_cast<float*>(raw + sizeof(Shared));
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const size_t row = blockIdx.x;
  const int V = p.V;
  const T* g = static_cast<const T*>(p.logits) + row * p.ld;
  const RowReader<T, NT, CACHE> x{g, cache};

  // ---- maximum (lowest index first) and candidates
  float m = -CUDART_INF_F;
  int im = 0x7fffffff;
  unsigned cand = 0;
  for (int i = tid; i < V; i += NT) {
    float v = Elem<T>::get(g[i]);
    if (!(v > -CUDART_INF_F)) v = -CUDART_INF_F;   // NaN as -infinity
    else ++cand;
    if (CACHE) cache[i] = v;
    if (v > m) { m = v; im = i; }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, m, o);
    const int oi = __shfl_xor_sync(0xffffffffu, im, o);
    if (om > m || (om == m && oi < im)) { m = om; im = oi; }
    cand += __shfl_xor_sync(0xffffffffu, cand, o);
  }
  if (tid == 0) { sh.n = 0; sh.fmax = -CUDART_INF_F; sh.imax = 0x7fffffff; }
  __shared__ float wm[32];
  __shared__ int wi[32];
  if (lane == 0) { wm[warp] = m; wi[warp] = im; }
  __syncthreads();
  if (lane == 0) atomicAdd(&sh.n, cand);
  if (tid == 0)
    for (int w = 0; w < NT / 32; ++w)
      if (wm[w] > sh.fmax || (wm[w] == sh.fmax && wi[w] < sh.imax)) {
        sh.fmax = wm[w];
        sh.imax = wi[w];
      }
  __syncthreads();
  const float top = sh.fmax;
  const int ncand = (int)sh.n;
  const float temp = p.temperature ? p.temperature[row] : p.temperature0;
  if (ncand == 0 || !(temp > 0.f)) {
    if (tid == 0) p.out[row] = ncand == 0 ? -1 : sh.imax;
    return;
  }
  const int k = p.top_k ? p.top_k[row] : p.top_k0;
  const float tp = p.top_p ? p.top_p[row] : p.top_p0;
  const double mp = fmin((double)(p.min_p ? p.min_p[row] : p.min_p0), 1.0);
  const double dtop = (double)top, dtemp = (double)temp, unit = exp2((double)p.shift);
  const float inv_t = 1.f / temp;

  auto weight = [&](float v) -> double {
    return v == top ? 1.0 : exp(((double)v - dtop) / dtemp);
  };
  auto units = [&](float v) -> u64 { return __double2ull_rn(weight(v) * unit); };
  // a bin of the order: monotone in v, equal values share it
  auto bin_of = [&](float v) -> int {
    const float d = (top - v) * inv_t * kBinsPerUnit;
    return v == top ? 0 : d < (float)(kBins - 1) ? (int)d : kBins - 1;
  };

  Cut cut;
  // The cut of the shortest prefix (of what `cut` keeps) whose measure reaches
  // thr: counts, or weights.  The histogram of level 0 is in sh.
  auto select = [&](bool mass, u64 thr) {
    find_bin<NT>(sh, mass, kBins, thr);
    const int bin = sh.found;
    u64 base = sh.found_base;
    unsigned prefix = 0;
    for (int level = 3; level >= 0; --level) {
      const int sft = level * 8;
      __syncthreads();
      for (int i = tid; i < 256; i += NT) { sh.count[i] = 0; sh.mass[i] = 0; }
      __syncthreads();
      for (int i = tid; i < V; i += NT) {
        const float v = x.at(i);
        if (!(v > -CUDART_INF_F) || bin_of(v) != bin) continue;
        const unsigned key = desc_key(v);
        if (!cut.has(key, i) || (level < 3 && (key >> (sft + 8)) != (prefix >> (sft + 8))))
          continue;
        atomicAdd(&sh.count[key >> sft & 255], 1u);
        if (mass) atomicAdd(&sh.mass[key >> sft & 255], units(v));
      }
      __syncthreads();
      find_bin<NT>(sh, mass, 256, thr - base);
      prefix |= (unsigned)sh.found << sft;
      base += sh.found_base;
    }
    // one value is left: the number of its ties to keep
    const unsigned ties = sh.count[prefix & 255];
    u64 need = thr - base;
    if (mass) {
      const u64 each = sh.mass[prefix & 255] / ties;
      need = (need + each - 1) / each;
    }
    Cut c;
    c.key = prefix;
    if (need < ties) {   // the need-th tie by index
      // warps own runs of indices
      const int seg = (V + NT / 32 - 1) / (NT / 32), s0 = warp * seg, s1 = min(s0 + seg, V);
      unsigned mine = 0;
      for (int i = s0 + lane; i - lane < s1; i += 32) {
        const bool t = i < s1 && x.at(i) > -CUDART_INF_F && desc_key(x.at(i)) == prefix &&
                       cut.has(prefix, i);
        mine += __popc(__ballot_sync(0xffffffffu, t));
      }
      __syncthreads();
      if (lane == 0) sh.wsum[warp] = mine;
      __syncthreads();
      u64 before = 0;
      for (int w = 0; w < warp; ++w) before += sh.wsum[w];
      if (before < need && before + mine >= need) {
        u64 left = need - before;
        for (int i = s0 + lane; i - lane < s1; i += 32) {
          const bool t = i < s1 && x.at(i) > -CUDART_INF_F && desc_key(x.at(i)) == prefix &&
                         cut.has(prefix, i);
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
    } else if (cut.key == prefix) {
      c.last = cut.last;
    }
    __syncthreads();
    cut = c;
  };
  auto clear = [&]() {
    __syncthreads();
    for (int i = tid; i < kBins; i += NT) { sh.count[i] = 0; sh.mass[i] = 0; }
    __syncthreads();
  };

  if (k > 0 && k < ncand) {
    clear();
    for (int i = tid; i < V; i += NT) {
      const float v = x.at(i);
      if (v > -CUDART_INF_F) atomicAdd(&sh.count[bin_of(v)], 1u);
    }
    __syncthreads();
    select(false, (u64)k);
  }
  if (tp < 1.f) {
    clear();
    u64 mine = 0;
    for (int i = tid; i < V; i += NT) {
      const float v = x.at(i);
      if (v > -CUDART_INF_F && cut.has(desc_key(v), i)) {
        const u64 w = units(v);
        mine += w;
        atomicAdd(&sh.mass[bin_of(v)], w);
      }
    }
    u64 total;
    block_prefix<NT>(mine, sh.wsum, &total);
    const double want = ceil((double)tp * (double)total);
    select(true, want >= 1.0 ? (u64)want : 1ull);   // NaN and p <= 0: the first token
  }

  // ---- draw: warps own runs of indices
  const int seg = (V + NT / 32 - 1) / (NT / 32), s0 = warp * seg, s1 = min(s0 + seg, V);
  auto kept = [&](int i) -> u64 {
    if (i >= s1) return 0;
    const float v = x.at(i);
    if (!(v > -CUDART_INF_F) || !cut.has(desc_key(v), i)) return 0;
    const double w = weight(v);
    return w >= mp ? __double2ull_rn(w * unit) : 0;
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
  const double at = (double)p.u[row] * (double)total;
  u64 thr = at > 0.0 ? (at < (double)total ? (u64)at + 1 : total) : 1;
  if (thr > total) thr = total;
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
  auto* kern = sample_kernel<T, NT, CACHE>;
  const int smem = (int)sizeof(Shared) + (CACHE ? p.V * 4 : 0);
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
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

cudaError_t launch_sample(const SampleParams& p, cudaStream_t s) {
  return p.dtype == M3_BF16 ? sample_rows<__nv_bfloat16>(p, s) : sample_rows<float>(p, s);
}

}  // namespace m3
