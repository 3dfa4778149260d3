// Launch interface of the sequence-model operators (norms, causal
// convolution, selective scan, token drawing) between their kernels and the C
// ABI.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace m3 {

constexpr int kMaxNormD = 32768;

struct NormParams {
  const void* x; long long ld_x;      // (rows, ld_x)
  const float* w; const float* b;     // (d,), b may be nullptr
  void* y;                            // (rows, d)
  float* mean; float* rstd;           // (rows,) or nullptr
  long long rows; int d;
  int dtype_x, dtype_y, rms;
  float eps;
  int sms;
};
cudaError_t launch_norm_fwd(const NormParams& p, cudaStream_t s);

struct NormBwdParams {
  const void* x; long long ld_x;
  const float* w;
  const float* mean; const float* rstd;
  const void* g;                      // (rows, d) of dtype_y
  void* dx;                           // (rows, d) of dtype_x
  float* dw; float* db;               // (d,), db may be nullptr
  float* part;                        // (norm_bwd_ctas, 2, d)
  long long rows; int d;
  int dtype_x, dtype_y, rms;
  int sms;
};
int norm_bwd_ctas(long long rows, int d, int sms);   // partials
cudaError_t launch_norm_bwd(const NormBwdParams& p, cudaStream_t s);

constexpr int kMaxConvWidth = 8;

struct ConvParams {
  const void* x; long long ld_x;      // (B*L, ld_x)
  const float* w; const float* b;     // (D, K), (D,) or nullptr
  const void* state;                  // (B, K-1, D): the rows before x, or nullptr (zeros)
  const int* lengths;                 // (B,) or nullptr
  void* y;                            // (B, L, D)
  void* state_out;                    // (B, K-1, D) or nullptr
  int B, L, D, K;
  int dtype, silu;
  int sms;
  int tt;                             // steps per thread, set by the launcher
};
cudaError_t launch_conv_fwd(const ConvParams& p, cudaStream_t s);

struct ConvBwdParams {
  const void* x; long long ld_x;
  const float* w; const float* b;
  const void* state; const int* lengths;
  const void* g;                      // (B, L, D)
  void* dx;                           // (B, L, D)
  float* dw; float* db;               // (D, K), (D,)
  float* part;                        // (workers, K + 1, D)
  int B, L, D, K;
  int dtype, silu;
  int sms;
  int workers, tt;                    // from conv_bwd_plan
};
void conv_bwd_plan(int B, int L, int D, int sms, int* workers, int* tt);
cudaError_t launch_conv_bwd(const ConvBwdParams& p, cudaStream_t s);

struct ConvStepParams {
  void* state;                        // (B, K-1, D), shifted in place
  const void* x; long long ld_x;      // (B, ld_x)
  const float* w; const float* b;
  void* y;                            // (B, D)
  int B, D, K;
  int dtype, silu;
};
cudaError_t launch_conv_step(const ConvStepParams& p, cudaStream_t s);

// Selective scan.  In the backward a lane group of `ln` threads shares a pair of
// channels, four states per thread and channel (the forward: half as many lanes,
// eight states each); NP = 4 * ln states are kept per channel.
constexpr int kMaxSelState = 128;
constexpr int kSelSteps = 16;         // steps staged at a time = checkpoint interval

inline int sel_lanes(int N) { return N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : N <= 64 ? 16 : 32; }
inline int sel_threads(int ln) { return ln >= 16 ? 256 : 128; }
inline int sel_tile(int ln) { return sel_threads(ln) / ln * 2; }   // channels per backward CTA

struct SelParams {
  const void* u; const void* dt; const void* z;          // (B*L, ld), z may be nullptr
  const void* Bm; const void* Cm;                        // (B*L, ld), N columns
  long long ld_u, ld_dt, ld_z, ld_b, ld_c;
  const float* A;                                        // (D, N)
  const float* dskip; const float* dt_bias;              // (D,) or nullptr
  const float* h0;                                       // (B, D, N) or nullptr
  const int* lengths;                                    // (B,) or nullptr
  void* y;                                               // (B, L, D)
  float* h_last;                                         // (B, D, N) or nullptr
  float* ckpt;                                           // (B, nch - 1, D, NP) or nullptr
  int B, L, D, N;
  int dtype, softplus;
  int nch;                                               // chunks of kSelSteps
  // time split: `splits` runs of cps chunks; each starts from hin (splits, B, D, NP),
  // which the summaries hsum (splits, B, D, NP) and dsum (splits, B, D) give
  int splits, cps;
  float* hin; float* hsum; float* dsum;
  int vec_d, vec_n;                                      // vector rows allowed
};
// CTAs per SM of the forward and the backward (0: error), channels per forward CTA.
int sel_fwd_resident(int N, int dtype);
int sel_bwd_resident(int N, int dtype);
inline int sel_fwd_tile(int N) { return N <= 8 ? 128 : 64; }
cudaError_t launch_sel_fwd(const SelParams& p, cudaStream_t s);

struct SelBwdParams {
  SelParams f;                                           // y unused
  const void* g;                                         // (B, L, D)
  void* du; void* ddt; void* dz;                         // (B, L, D)
  void* dB; void* dC;                                    // (B, L, N)
  float* dA; float* dD; float* dbias;                    // (D, N), (D,), (D,)
  int b0, nb;                                            // rows of a slab (launcher: the first)
  float* part_bc;                                        // (G, nb*L, 2, NP)
  float* part_a;                                         // (workers, D, NP + 2)
  int workers;                                           // CTAs along the batch and the splits
  int bgroups;                                           // workers / splits
  float* qin; float* qsum;                               // (splits, B, D, NP)
  int vec_g;
};
cudaError_t launch_sel_bwd(const SelBwdParams& p, cudaStream_t s);

struct SelStepParams {
  float* h;                                              // (B, D, N), updated in place
  const void* u; const void* dt; const void* z;          // (B, ld)
  const void* Bm; const void* Cm;                        // (B, ld)
  long long ld_u, ld_dt, ld_z, ld_b, ld_c;
  const float* A; const float* dskip; const float* dt_bias;
  void* y;                                               // (B, D)
  int B, D, N;
  int dtype, softplus;
};
cudaError_t launch_sel_step(const SelStepParams& p, cudaStream_t s);

constexpr int kMaxVocab = 1 << 18;

struct SampleParams {
  const void* logits; long long ld;                      // (rows, ld)
  const float* u;                                        // (rows,)
  // per-row settings, or nullptr: the scalars
  const float* temperature; const int* top_k; const float* top_p; const float* min_p;
  float temperature0, top_p0, min_p0; int top_k0;
  long long* out;                                        // (rows,)
  int rows, V, dtype;
  int shift;                                             // weights in units of 2^-shift
  int sms;
  int vec;                                               // 16-byte loads, set by the launcher
};
cudaError_t launch_sample(const SampleParams& p, cudaStream_t s);

}  // namespace m3
