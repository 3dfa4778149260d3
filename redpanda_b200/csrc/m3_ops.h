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

// RMS norm of the residual stream with the branch's addition: s = x + res.
struct AddNormParams {
  const void* x; long long ld_x;      // (rows, ld_x), the branch
  const void* res; long long ld_r;    // (rows, ld_r), the stream
  const float* w;                     // (d,)
  void* y;                            // (rows, d)
  void* s;                            // (rows, d) of the stream's type
  float* rstd;                        // (rows,) or nullptr
  long long rows; int d;
  int dtype_x, dtype_s, dtype_y;
  float eps;
  int sms;
};
cudaError_t launch_add_norm_fwd(const AddNormParams& p, cudaStream_t s);

struct AddNormBwdParams {
  const void* s; long long ld_s;      // (rows, ld_s)
  const float* w; const float* rstd;
  const void* gy;                     // (rows, d) of dtype_y
  const void* gs;                     // (rows, d) of dtype_s or nullptr: zero
  void* ds;                           // (rows, d) of dtype_s
  void* dx;                           // (rows, d) of dtype_x, or nullptr: ds serves
  float* dw;                          // (d,)
  float* part;                        // (add_norm_bwd_ctas, d)
  long long rows; int d;
  int dtype_x, dtype_s, dtype_y;
  int sms;
};
int add_norm_bwd_ctas(long long rows, int d, int sms);   // partials
cudaError_t launch_add_norm_bwd(const AddNormBwdParams& p, cudaStream_t s);
// out[c] = sum over n partials part[(i * arrays + which) * d + c], which: 0 for dw, 1 for db,
// in a fixed order (db may be nullptr)
cudaError_t launch_norm_reduce(const float* part, int n, int d, int arrays, float* dw, float* db,
                               cudaStream_t s);

// The RMS norm (of x, or of s = x + res) in 8 bits with scales.
struct Norm8Params {
  const void* x; long long ld_x;      // (rows, ld_x)
  const void* res; long long ld_r;    // (rows, ld_r) of dtype_s, or nullptr
  const float* w;                     // (d,)
  unsigned char* q;                   // (rows, d)
  float* scale;                       // (rows, d / group), or (rows,) for group 0
  void* s;                            // (rows, d) of dtype_s, unused without res
  long long rows; int d, group;
  int dtype_x, dtype_s;
  int e4m3;                           // else int8
  float eps;
  int sms;
};
cudaError_t launch_norm8(const Norm8Params& p, cudaStream_t s);

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

// Gated linear recurrence: see m3_gated.cuh.
struct GatedParams {
  const void* x; const void* rg; const void* ig;         // (B*L, ld)
  long long ld_x, ld_r, ld_i;
  const float* decay; float c;                           // (D,)
  const float* h0;                                       // (B, D) or nullptr
  const int* lengths;                                    // (B,) or nullptr
  void* y;                                               // (B, L, D)
  float* h_last;                                         // (B, D) or nullptr
  float* ckpt;                                           // (B, segments, D) or nullptr
  int B, L, D;
  int dtype;
  int lanes, warps, splits, rows;                        // per run, per CTA, per cluster; grid
  int solo;                                              // a warp walks its rows by itself
  int copy;                                              // how rows are copied (m3_gated.cuh)
  int* err;                                              // the device's error word
};
struct GatedBwdParams {
  GatedParams f;                                         // y, h_last unused
  const void* g;                                         // (B, L, D)
  void* dx; void* drg; void* dig;                        // (B, L, D)
  float* ddecay;                                         // (D,)
  float* part;                                           // (rows * splits, D)
};
int gated_segments(int L);                               // checkpoints per row and channel
// sets lanes, warps, splits and rows
void gated_plan(int B, int L, int D, bool backward, int sms, GatedParams* p);
int gated_bwd_in_clusters(int k);                        // the backward's CTAs resident in clusters of k
cudaError_t launch_gated_fwd(const GatedParams& p, cudaStream_t s);
cudaError_t launch_gated_bwd(const GatedBwdParams& p, cudaStream_t s);

struct GatedStepParams {
  float* h;                                              // (B, D), updated in place
  const void* x; const void* rg; const void* ig;         // (B, ld)
  long long ld_x, ld_r, ld_i;
  const float* decay; float c;
  void* y;                                               // (B, D)
  int B, D, dtype, sms;
};
cudaError_t launch_gated_step(const GatedStepParams& p, cudaStream_t s);

// Product of a few rows with 4-bit weights (m3_gemv4.cu).
constexpr int kQ4Rows = 8;
constexpr int kQ4MaxIn = 65536;
struct RowsQ4Params {
  const void* x; long long ld_x;                         // (rows, d_in)
  const float* norm_w; float eps;                        // RMS norm weight or nullptr
  const uint4* codes;                                    // (tiles, blocks, 32): see m3_gemv4.cu
  const void* scales;                                    // (tiles, groups, 8) words
  const float* bias;                                     // (d_out,) or nullptr
  const void* residual; long long ld_r;                  // (rows, d_out) or nullptr
  void* out0; long long ld0;
  void* out1; long long ld1;
  int rows, d_in, d_out, split, silu, group, center, dtype;
  int pdl, sms;
  int vec, vec8;                                         // x and norm_w in vectors of 4; bf16 x in vectors of 8 (2), words (1) or not
  int mw, kw, chunk;                                     // set by the launcher
};
cudaError_t launch_rows_q4(const RowsQ4Params& p, cudaStream_t s);

}  // namespace m3
