/*
 * m3scan.h - C ABI of the B200 (sm_100a) Mamba-3 trapezoidal selective scan.
 *
 * Drop-in kernels for the hot path of PranavPrasannaV/RedPanda's Mamba-3
 * backbone.  Every entry point takes plain device pointers, sizes and a CUDA
 * stream (passed as void*), returns 0 or an M3_ERR_* code, never throws,
 * never allocates and never frees: the caller owns every input, output and
 * workspace buffer.  All pointers are device pointers to dense, row-major
 * (contiguous) tensors.
 *
 * Interface map (reference file:line -> entry point):
 *   redpanda/engine/triton_scan.py:248-281  _TrapezoidalScanFn.forward  -> m3_scan_fwd
 *   redpanda/engine/triton_scan.py:283-315  _TrapezoidalScanFn.backward -> m3_scan_bwd
 *   redpanda/engine/mamba.py:254-260        bidirectional scan pair     -> m3_scan_fwd/bwd with
 *                                                                          M3_DIR_BIDIR
 *   redpanda/engine/mamba.py:343,377-379    return_state (h_last, dBu_last) -> m3_scan_fwd h_last/dbu_last
 *   redpanda/engine/mamba.py:466-493        Mamba3Block.step recurrence -> m3_step
 *   redpanda/engine/mamba.py:455-469        step inputs (softplus, BCNorm, MIMO fold) -> m3_step_inputs
 *   redpanda/engine/mamba.py:490-497        step + gated output (y + u*D) * silu(z) -> m3_step_gated
 *   redpanda/engine/mamba.py:455-497        step inputs + step + gated output in one launch
 *                                           -> m3_step_gated_fused (+ dt_proj: _proj)
 *   redpanda/engine/mamba.py:262-265        (y + u*D) * silu(z) after a scan -> m3_gate
 *                                           and its autograd backward -> m3_gate_bwd
 *   redpanda/engine/mamba.py:243, 452       u = silu(x half of in_proj) -> m3_silu
 *   redpanda/engine/mamba.py:82-89, 450-452 RMSNorm + in_proj + silu, small batch -> m3_rows_linear
 *   redpanda/engine/mamba.py:454, 463       x_proj + dt_proj product, small batch -> m3_xdt_proj
 *   redpanda/engine/mamba.py:497, 591-595   out_proj + residual add, small batch -> m3_rows_linear
 *   redpanda/engine/mamba.py:82-89          RMSNorm, forward and backward -> m3_norm_fwd / m3_norm_bwd
 *
 * Shapes (B batch, L length, D = d_inner, N = d_state, n_rot rotational lanes,
 * N - n_rot tracking lanes):
 *   delta, u            (B, L, D)  dtype_du  (post-softplus delta, SSM input)
 *   Bc, Cc              (B, L, N)  dtype_bc  (MIMO-contracted, BCNorm'ed B and C)
 *   A_real_p, A_imag_p  (D, N)     float32   rotational eigenvalues in columns
 *                                            [0, n_rot), zero elsewhere
 *   track_p             (D, N)     float32   tanh(theta) in columns [n_rot, N)
 *   (the padded parameter layout of triton_scan.py:325-335)
 *   y                   (B, L, D)  float32   scan output WITHOUT the u*D skip
 */
#ifndef M3SCAN_H
#define M3SCAN_H

#include <stddef.h>
#include <stdint.h>

#if defined(__GNUC__)
#define M3_API __attribute__((visibility("default")))
#else
#define M3_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

/* element types */
enum { M3_F32 = 0, M3_BF16 = 1 };

/* scan directions.  M3_DIR_REV scans the sequence back to front, which equals
 * flip(scan(flip(x))) of the reference (mamba.py:258-260); M3_DIR_BIDIR writes
 * y_fwd + y_rev in one launch. */
enum { M3_DIR_FWD = 0, M3_DIR_REV = 1, M3_DIR_BIDIR = 2 };

/* status codes */
enum {
  M3_OK = 0,
  M3_ERR_NULL = 1,         /* a required pointer is NULL */
  M3_ERR_SHAPE = 2,        /* a size is out of range */
  M3_ERR_DTYPE = 3,        /* unsupported element type */
  M3_ERR_UNSUPPORTED = 4,  /* no compiled kernel serves this shape (a (d_state, n_rot)
                              split, or a size past a kernel's stated limit) */
  M3_ERR_ALIGN = 5,        /* a pointer is not aligned to its element size */
  M3_ERR_WORKSPACE = 6,    /* workspace missing or too small */
  M3_ERR_LAUNCH = 7,       /* the CUDA launch failed (see cudaGetLastError) */
  M3_ERR_DEVICE = 8,       /* a kernel recorded a device-side error */
  M3_ERR_NO_DEVICE = 9,    /* no CUDA device / the current device is not sm_100 */
  M3_ERR_SCRATCH_LIMIT = 10, /* m3_scan_bwd_noalloc: the problem needs more scratch than
                                M3_NOALLOC_SCRATCH_BYTES */
  M3_ERR_ALIAS = 11          /* two buffers that must be distinct overlap */
};

typedef struct m3_scan_desc {
  int32_t batch;      /* B >= 1 */
  int32_t seqlen;     /* L >= 1 */
  int32_t d_inner;    /* D >= 1 */
  int32_t d_state;    /* N, 1..128 */
  int32_t n_rot;      /* 0..N rotational lanes; N - n_rot tracking lanes */
  int32_t dtype_du;   /* element type of delta and u (M3_F32 or M3_BF16) */
  int32_t dtype_bc;   /* element type of Bc and Cc */
  int32_t direction;  /* M3_DIR_FWD, M3_DIR_REV or M3_DIR_BIDIR */
} m3_scan_desc;

typedef struct m3_step_desc {
  int32_t batch;      /* rows advanced in lockstep */
  int32_t d_inner;
  int32_t d_state;
  int32_t n_rot;
  int32_t dtype_du;
  int32_t dtype_bc;
} m3_step_desc;

/* Human-readable text of a status code (static storage). */
M3_API const char* m3_strerror(int code);

/* ABI version: (major << 16) | minor. */
M3_API int m3_version(void);

/* Number of float32 elements of the forward checkpoint buffer the backward
 * consumes: the state every 8 steps for the (16 rotational + 16 tracking)
 * lane layout, every 16 steps otherwise; 0 when L fits one interval.  The
 * buffer must be 16-byte aligned.  Replaces the hck/dck chunk checkpoints that
 * triton_scan.py:261-262 allocates. */
M3_API size_t m3_scan_ckpt_floats(const m3_scan_desc* desc);

/* Forward scan.  Replaces _TrapezoidalScanFn.forward (triton_scan.py:248-281)
 * and the return_state branch of _selective_scan_trapezoidal (mamba.py:377-379).
 *   y         required, (B, L, D) float32
 *   ckpt      optional (NULL = inference only); m3_scan_ckpt_floats() floats,
 *             16-byte aligned, to be handed to m3_scan_bwd
 *   h_last,   optional, (B, D, N) float32: state after the last token of the
 *   dbu_last  scan direction (M3_DIR_FWD or M3_DIR_REV only) */
M3_API int m3_scan_fwd(const m3_scan_desc* desc,
                const void* delta, const void* u, const void* Bc, const void* Cc,
                const float* A_real_p, const float* A_imag_p, const float* track_p,
                float* y, float* ckpt, float* h_last, float* dbu_last,
                void* stream);

/* m3_scan_fwd with the element type of y chosen by dtype_y (M3_F32 or
 * M3_BF16); the state and every accumulation stay fp32 and only the stored y
 * is rounded.  Replaces the same _TrapezoidalScanFn.forward
 * (triton_scan.py:248-281) for a bf16 layer (the reference's autocast
 * training, train.py:268, and the bf16 Eval-Mamba forward of model.py:110-132).
 * With M3_DIR_BIDIR and a bf16 y the first direction's partial is stored in
 * bf16 and the second adds to it in fp32 before rounding again (at most one
 * bf16 ulp more than a single rounding). */
M3_API int m3_scan_fwd_typed(const m3_scan_desc* desc,
                const void* delta, const void* u, const void* Bc, const void* Cc,
                const float* A_real_p, const float* A_imag_p, const float* track_p,
                void* y, int32_t dtype_y, float* ckpt, float* h_last, float* dbu_last,
                void* stream);

/* Forward scan with the layer's prologue fused into its staging
 * (mamba.py:284-301 and 336-337, the projections' softplus, BCNorm and MIMO
 * fold that otherwise run before the scan).  bf16 inputs only (the
 * config-1/2 element types; desc->dtype_du must be M3_BF16, dtype_bc is
 * ignored):
 *   dt      (B, L, D) bf16: dt_proj output including its bias, before softplus
 *   xbc     (B*L, ld_x) bf16: x_proj output rows; B_raw = columns
 *           [off_b, off_b + N*mimo_p), C_raw = [off_c, off_c + N*mimo_p)
 *   wb, wc  (N*mimo_p,) float32 BCNorm weights, or both NULL (use_bcnorm=False)
 *   u       (B, L, D) bf16
 * The scan sees delta = bf16(softplus(dt)) and Bc, Cc = bf16 of the fold of
 * BCNorm(B_raw), BCNorm(C_raw) (computed in fp32 as m3_step_inputs does), so
 * y and ckpt equal those of m3_step_inputs + casts to bf16 + m3_scan_fwd_typed
 * bit for bit.  Shapes the staging cannot take (column offsets off 8-element
 * boundaries, N*mimo_p above 256, channel counts off the tile) return
 * M3_ERR_UNSUPPORTED: run the unfused pair then. */
M3_API int m3_scan_fwd_fused(const m3_scan_desc* desc, int32_t mimo_p, const void* dt,
                const void* xbc, int64_t ld_x, int32_t off_b, int32_t off_c,
                const float* wb, const float* wc, float eps, const void* u,
                const float* A_real_p, const float* A_imag_p, const float* track_p,
                void* y, int32_t dtype_y, float* ckpt, void* stream);

/* Workspace bytes m3_scan_bwd needs on the current device. */
M3_API size_t m3_scan_bwd_workspace_bytes(const m3_scan_desc* desc);

/* Analytic backward.  Replaces _TrapezoidalScanFn.backward
 * (triton_scan.py:283-315) with deterministic reductions (no atomics).
 *   dy        (B, L, D) of dtype_dy, the gradient of y
 *   ckpt      the forward's checkpoint buffer (NULL allowed when
 *             m3_scan_ckpt_floats() is 0)
 *   d_delta, d_u   (B, L, D) of dtype_du
 *   d_Bc, d_Cc     (B, L, N) of dtype_bc
 *   d_A_real_p, d_A_imag_p, d_track_p   (D, N) float32 in the padded layout
 *   workspace      >= m3_scan_bwd_workspace_bytes(desc) bytes */
M3_API int m3_scan_bwd(const m3_scan_desc* desc,
                const void* delta, const void* u, const void* Bc, const void* Cc,
                const float* A_real_p, const float* A_imag_p, const float* track_p,
                const void* dy, int32_t dtype_dy, const float* ckpt,
                void* d_delta, void* d_u, void* d_Bc, void* d_Cc,
                float* d_A_real_p, float* d_A_imag_p, float* d_track_p,
                void* workspace, size_t workspace_bytes, void* stream);

/* Workspace bytes of m3_scan_bwd_fused on the current device. */
M3_API size_t m3_scan_bwd_fused_workspace_bytes(const m3_scan_desc* desc, int32_t mimo_p);

/* Analytic backward of m3_scan_fwd_fused: the scan's backward with the
 * prologue's backward fused in (the gradients torch's softplus, RMSNorm and
 * sum give for mamba.py:284-301 and 336-337).  Inputs as m3_scan_fwd_fused,
 * plus dy (B, L, D) of dtype_dy and the forward's ckpt.  Outputs:
 *   d_dt    (B, L, D) bf16: softplus'(dt) times the bf16-rounded d delta
 *   d_u     (B, L, D) bf16
 *   d_xbc   (B*L, ld_x) bf16: the B_raw and C_raw columns are written; the
 *           caller zero-fills the rest (the dt_raw columns get their gradient
 *           through dt_proj)
 *   d_wb, d_wc (N*mimo_p,) float32 BCNorm weight gradients (fixed-order sums)
 *   d_A_real_p, d_A_imag_p, d_track_p  as m3_scan_bwd
 * Every output equals, bit for bit, what the unfused bf16 layer's backward
 * (m3_scan_bwd on the bf16 delta/Bc/Cc, then m3_step_inputs_bwd on the fp32
 * values of their bf16 gradients) produces. */
M3_API int m3_scan_bwd_fused(const m3_scan_desc* desc, int32_t mimo_p, const void* dt,
                const void* xbc, int64_t ld_x, int32_t off_b, int32_t off_c,
                const float* wb, const float* wc, float eps, const void* u,
                const float* A_real_p, const float* A_imag_p, const float* track_p,
                const void* dy, int32_t dtype_dy, const float* ckpt, void* d_dt, void* d_u,
                void* d_xbc, float* d_wb, float* d_wc, float* d_A_real_p, float* d_A_imag_p,
                float* d_track_p, void* workspace, size_t workspace_bytes, void* stream);

/* O(1) recurrent step of B rows, in place.  Replaces the recurrence of
 * Mamba3Block.step (mamba.py:466-493):
 *   h, dbu    (B, D, N) float32, read and overwritten with the new state
 *   delta, u  (B, D) of dtype_du;  Bc, Cc  (B, N) of dtype_bc
 *   y         (B, D) float32, sum_n h*C without the u*D skip
 * Bit-identical to m3_scan_fwd (M3_DIR_FWD) at every position when fed the
 * same per-token inputs and the scan's state. */
M3_API int m3_step(const m3_step_desc* desc, float* h, float* dbu,
            const void* delta, const void* u, const void* Bc, const void* Cc,
            const float* A_real_p, const float* A_imag_p, const float* track_p,
            float* y, void* stream);

/* O(1) step with the factored state: the same recurrence as m3_step with half
 * its HBM traffic.  The state is h (B, D, N) fp32, updated in place, and the
 * factors of the last token's input contribution, fac (B, D + N) fp32 =
 * [delta*u (D) | B (N)], read from fac_prev and written to fac_next (distinct
 * buffers; swap them between steps).  dBu = (delta*u)*B is rebuilt with the
 * scan's own rounding, so the outputs equal m3_step's bit for bit.  The
 * factors after a scan are [delta[L-1]*u[L-1] | Bc[L-1]] of its inputs.
 * Extends the cache contract of Mamba3Block.step (mamba.py:487-498), whose
 * dBu tensor it replaces by its two factors. */
M3_API int m3_step_factored(const m3_step_desc* desc, float* h, const float* fac_prev,
            float* fac_next, const void* delta, const void* u, const void* Bc, const void* Cc,
            const float* A_real_p, const float* A_imag_p, const float* track_p,
            float* y, void* stream);

/* The per-token step inputs from the layer's projection outputs, in one launch.
 * Replaces the elementwise part of Mamba3Block.step (mamba.py:455-469):
 *   delta (B, D)  = softplus(dt), torch's threshold 20
 *   Bc, Cc (B, N) = sum over the p MIMO columns of BCNorm(B_raw), BCNorm(C_raw)
 * with BCNorm(x) = x * rsqrt(mean(x^2) + eps) * w over the N*p vector
 * (mamba.py:82-89, 297-299, 336-337).
 *   dt      (B, ld_dt) desc->dtype_du: dt_proj(dt_raw), with its bias or without it
 *   dt_bias (D,) float32 dt_proj bias, added to dt first (one fp32 rounding, as
 *           torch's matmul-then-add), or NULL when dt includes it
 *   xbc     (B, ld_x) desc->dtype_bc: rows of x_proj's output; B_raw starts at
 *           column off_b and C_raw at off_c, N*p columns each
 *   wb, wc  (N*p,) float32 BCNorm weights, or both NULL (use_bcnorm=False: plain sum)
 *   delta   (B, D) desc->dtype_du; Bc, Cc (B, N) desc->dtype_bc
 * Arithmetic is fp32; a bf16 output is rounded once (the bits of the fp32
 * result cast to bf16, as a bf16 layer's casts give).  desc->n_rot is ignored. */
M3_API int m3_step_inputs(const m3_step_desc* desc, int32_t mimo_p,
            const void* dt, int64_t ld_dt, const float* dt_bias, const void* xbc,
            int64_t ld_x, int32_t off_b, int32_t off_c, const float* wb, const float* wc,
            float eps, void* delta, void* Bc, void* Cc, void* stream);

/* u = silu(x) = x / (1 + exp(-x)) over (rows, d) of a row-strided x: the x half
 * of in_proj's output (mamba.py:243, 452), read in place; out (rows, d) float32
 * contiguous. */
M3_API int m3_silu(int64_t rows, int32_t d, const float* x, int64_t ld_x, float* out,
            void* stream);

/* Small-batch projections of the step layer (at most 8 rows; a search node or
 * a few lines), fp32, for the launch-latency-bound regime where each
 * projection is a matrix-vector product.  One warp per output column; sums in
 * a fixed order (deterministic); weights (nn.Linear layout, (d_out, d_in)
 * row-major) 16-byte aligned with d_in % 4 == 0.  rows > 8, or inputs past 48 KB
 * of staged floats (8 rows x 1536, 2 x 6144, ...), return M3_ERR_UNSUPPORTED.
 *
 * m3_rows_linear: out = act(residual + (bias + xn W^T)) with
 *   xn = x * rsqrt(mean(x^2) + eps) * norm_w    (RMSNorm, mamba.py:82-89) when
 *        norm_w != NULL, else x;
 *   columns [0, split) -> out0 (row stride ld0), silu applied when silu != 0
 *        (the x half of in_proj, mamba.py:450-452); columns [split, d_out) ->
 *        out1 (row stride ld1; the z half);
 *   residual (rows, ld_r) or NULL, added last (mamba.py:595); it may be out0
 *        itself (out_proj + residual in place), but no output may overlap x
 *        (M3_ERR_ALIAS).
 * Rounding differs from a cuBLAS GEMM only by the summation order.
 *
 * overlap != 0 (here, in m3_xdt_proj and in m3_step_gated_fused_proj): launch
 * as a programmatic dependent launch, so that the kernel starts while the one
 * ahead of it on the stream finishes (a chain of these calls, as one step
 * layer makes, then pays one launch latency instead of one per call).
 * m3_rows_linear reads the first part of its weight rows W before that kernel
 * has completed: set overlap only when no kernel queued before the call
 * writes W.  Everything else is read after it has completed. */
M3_API int m3_rows_linear(int32_t rows, int32_t d_in, int32_t d_out, const float* x,
            int64_t ld_x, const float* norm_w, float eps, const float* W,
            const float* bias, const float* residual, int64_t ld_r, int32_t split,
            int32_t silu, float* out0, int64_t ld0, float* out1, int64_t ld1,
            int32_t overlap, void* stream);

typedef struct m3_rows_q4_desc {
  int32_t rows;       /* 1..8 */
  int32_t d_in;       /* 1..65536 */
  int32_t d_out;      /* >= 1 */
  int32_t group;      /* columns per scale: 32, 64 or 128 */
  int32_t center;     /* non-zero: a center beside each scale */
  int32_t dtype;      /* element type of x, residual, out0 and out1 */
  int32_t split;      /* columns of out0 */
  int32_t silu;       /* non-zero: silu on the columns of out0 */
  float eps;          /* of the norm */
} m3_rows_q4_desc;

/* m3_rows_linear with weights of 4 bits: out = act(residual + (bias + xn W^T)),
 *   W[o,k] = scale[o,k/group] (q[o,k] - 8) + center[o,k/group],  q in 0..15,
 * in fp32 (inputs are not rounded), each output rounded once; the norm, split,
 * residual and overlap as above (the codes and scales are the weights that overlap
 * is about).  Sums in a fixed order; scale and center come in behind a group's sums,
 * so a row with an infinity, or past 1e35, may give NaN.
 *   codes   (tiles, blocks, 32, 4) 32-bit words, 16-byte aligned: tiles of 16
 *           outputs, blocks of 64 columns; both numbers rounded up, the columns to
 *           whole groups of 128 where group is 128.  Word j of lane l of a block
 *           holds, in bits 4 (h + 2 v + 4 e) up, the code of output l / 4 + 8 h and
 *           column 32 (j / 2) + 8 (l % 4) + 4 (j % 2) + 2 v + e (h, v, e: 0, 1).
 *   scales  (tiles, groups, 8) of two outputs each, l and l + 8: bf16 pairs of
 *           scale and center (64 bits) with center, else their two scales (32
 *           bits); 16-byte aligned; groups cover the rounded-up columns
 *   x (rows, ld_x); norm_w (d_in,) float32 or NULL; bias (d_out,) float32 or NULL;
 *   residual (rows, ld_r) or NULL: it may be out0 itself (same stride, split ==
 *   d_out), no other overlap of an output with an input; out0 and out1 may be
 *   columns of one buffer, but share no element (M3_ERR_ALIAS). */
M3_API int m3_rows_linear_q4(const m3_rows_q4_desc* desc, const void* x, int64_t ld_x,
            const float* norm_w, const void* codes, const void* scales, const float* bias,
            const void* residual, int64_t ld_r, void* out0, int64_t ld0, void* out1, int64_t ld1,
            int32_t overlap, void* stream);

/* m3_xdt_proj: x_dbl = u W_x^T + b_x  (rows, n_x; mamba.py:454) and
 * dt = x_dbl[:, :dt_rank] W_dt^T  (rows, d_inner; dt_proj without its bias,
 * mamba.py:463 -- m3_step_gated_fused / m3_step_inputs add it) in one launch.
 * u (rows, d_inner) contiguous; W_x (n_x, d_inner); b_x (n_x,) or NULL; W_dt
 * (d_inner, dt_rank), dt_rank <= 64 (else M3_ERR_UNSUPPORTED).  u, x_dbl and dt
 * must not overlap. */
M3_API int m3_xdt_proj(int32_t rows, int32_t d_inner, int32_t n_x, int32_t dt_rank,
            const float* u, const float* W_x, const float* b_x, const float* W_dt,
            float* x_dbl, float* dt, int32_t overlap, void* stream);

/* Workspace bytes of m3_step_inputs_bwd (the BCNorm weight-gradient partials). */
M3_API size_t m3_step_inputs_bwd_workspace_bytes(const m3_step_desc* desc, int32_t mimo_p);

/* Backward of m3_step_inputs over desc->batch rows (the training-path prologue:
 * the gradients that torch's softplus, RMSNorm and sum backward give for
 * mamba.py:284-301 and 336-337):
 *   dt, g_delta, d_dt       (rows, D) of desc->dtype_du; d_dt = g_delta * softplus'(dt)
 *   xbc, d_xbc              (rows, ld_x) of desc->dtype_bc: columns [off_b, off_b + N*p)
 *                           and [off_c, off_c + N*p) of d_xbc are written (the gradients
 *                           of B_raw, C_raw); other columns are left untouched
 *   g_Bc, g_Cc              (rows, N) of desc->dtype_bc: upstream gradients
 *   d_wb, d_wc (N*p,) float32 BCNorm weight gradients, reduced over the rows in a
 *           fixed order (bitwise reproducible); unused when wb == wc == NULL
 *   workspace >= m3_step_inputs_bwd_workspace_bytes(desc, mimo_p) bytes
 * Arithmetic is fp32; bf16 gradients are rounded once. */
M3_API int m3_step_inputs_bwd(const m3_step_desc* desc, int32_t mimo_p,
            const void* dt, int64_t ld_dt, const void* xbc, int64_t ld_x,
            int32_t off_b, int32_t off_c, const float* wb, const float* wc, float eps,
            const void* g_delta, const void* g_Bc, const void* g_Cc,
            void* d_dt, void* d_xbc, float* d_wb, float* d_wc,
            void* workspace, size_t workspace_bytes, void* stream);

/* m3_step (dbu != NULL) or m3_step_factored (fac_prev, fac_next != NULL, dbu
 * NULL) whose output is the layer's gated activation instead of y
 * (mamba.py:493-497):
 *   out (B, D) float32 = (y + u * d_skip) * silu(z),   silu(z) = z / (1 + exp(-z))
 *   z       (B, ld_z) float32: the z half of in_proj's output (before silu)
 *   d_skip  (D,) float32: the layer's skip weight D
 * The state update is identical to m3_step / m3_step_factored. */
M3_API int m3_step_gated(const m3_step_desc* desc, float* h, float* dbu,
            const float* fac_prev, float* fac_next, const void* delta, const void* u,
            const void* Bc, const void* Cc, const float* A_real_p, const float* A_imag_p,
            const float* track_p, const float* z, int64_t ld_z, const float* d_skip,
            float* out, void* stream);

/* m3_step_gated with the step's prologue in the same launch (mamba.py:455-497:
 * softplus(dt_proj), BCNorm of B_raw / C_raw, the MIMO fold, the recurrence and
 * the gated output): the kernel stages each row's dt and raw x_proj rows and
 * computes delta, Bc and Cc itself with the arithmetic of m3_step_inputs, so
 * the state and out are bit-identical to m3_step_inputs followed by
 * m3_step_gated.
 *   dt      (B, ld_dt) float32: dt_proj output, before softplus; dt_bias (D,) or
 *           NULL as for m3_step_inputs
 *   xbc     (B, ld_x) float32: x_proj output; B_raw at column off_b, C_raw at
 *           off_c, N * mimo_p values each
 *   wb, wc  (N * mimo_p,) float32 BCNorm weights, or both NULL (plain fold)
 *   u       (B, D) of desc->dtype_du; desc->dtype_bc must be M3_F32
 * Served by the pipelined step kernel for dense 32-lane states (N = 32, no
 * virtual lanes) with D % 32 == 0, mimo_p <= 2, and 16-byte aligned rows of dt,
 * xbc (ld_x, off_b, off_c multiples of 4), u and the state; any other shape
 * returns M3_ERR_UNSUPPORTED with nothing launched (run m3_step_inputs and
 * m3_step_gated instead). */
M3_API int m3_step_gated_fused(const m3_step_desc* desc, int32_t mimo_p, float* h, float* dbu,
            const float* fac_prev, float* fac_next, const float* dt, int64_t ld_dt,
            const float* dt_bias, const float* xbc, int64_t ld_x, int32_t off_b, int32_t off_c,
            const float* wb, const float* wc, float eps, const void* u,
            const float* A_real_p, const float* A_imag_p, const float* track_p,
            const float* z, int64_t ld_z, const float* d_skip, float* out, void* stream);

/* m3_step_gated_fused with dt_proj's product formed in the kernel too:
 * dt = xbc[:, :dt_rank] W_dt^T (mamba.py:463, the dt_raw columns of x_proj's
 * output times dt_proj's weight, W_dt (D, dt_rank) row-major float32,
 * dt_rank <= 64), then delta = softplus(dt + dt_bias) and the rest as
 * m3_step_gated_fused.  One launch for the whole step after x_proj; the dt sum
 * runs in a fixed order (4 strided partials, then pairs), so results are
 * deterministic but not the bits of a cuBLAS dt_proj. */
M3_API int m3_step_gated_fused_proj(const m3_step_desc* desc, int32_t mimo_p, float* h,
            float* dbu, const float* fac_prev, float* fac_next, const float* W_dt,
            int32_t dt_rank, const float* dt_bias, const float* xbc, int64_t ld_x,
            int32_t off_b, int32_t off_c, const float* wb, const float* wc, float eps,
            const void* u, const float* A_real_p, const float* A_imag_p,
            const float* track_p, const float* z, int64_t ld_z, const float* d_skip,
            float* out, int32_t overlap, void* stream);

/* The layer's gated activation after a scan (mamba.py:262-265), elementwise
 * over (rows, D) = (B*L, D):
 *   out = (y + coef * (u * d_skip)) * silu(z),   silu(z) = z / (1 + exp(-z))
 *   y (rows, D) float32 scan output; u (rows, D) of dtype_u (the SSM input);
 *   z (rows, ld_z) float32, the z half of in_proj's output; d_skip (D,) float32;
 *   coef 1 for one direction, 2 for the bidirectional pair (which adds u*D once
 *   per direction, mamba.py:256-260).  out may equal y (in place). */
M3_API int m3_gate(int64_t rows, int32_t d_inner, const float* y, const void* u,
            int32_t dtype_u, const float* z, int64_t ld_z, const float* d_skip, float coef,
            float* out, void* stream);

/* m3_gate with an element type per operand (M3_F32 or M3_BF16): y, u, z and
 * out of a bf16 layer (mamba.py:262-265 under the reference's autocast,
 * train.py:268; the bf16 Eval-Mamba forward, model.py:110-132).  Arithmetic is
 * fp32; out is rounded once.  out may equal y only when dtype_out == dtype_y.
 * round_silu != 0 rounds silu(z) to bf16 when z is bf16, as torch's F.silu on a
 * bf16 tensor does before the product (the training path's autograd formula,
 * mamba.py:265). */
M3_API int m3_gate_typed(int64_t rows, int32_t d_inner, const void* y, int32_t dtype_y,
            const void* u, int32_t dtype_u, const void* z, int32_t dtype_z, int64_t ld_z,
            const float* d_skip, float coef, int32_t round_silu, void* out, int32_t dtype_out,
            void* stream);

/* Workspace bytes of m3_gate_bwd (the per-row-chunk partial sums of d d_skip). */
M3_API size_t m3_gate_bwd_workspace_bytes(int64_t rows, int32_t d_inner);

/* Backward of m3_gate_typed (the autograd of mamba.py:262-265 / 496-497 in one
 * launch plus a fixed-order reduction): with a = y + coef*u*d_skip,
 * s = silu(z) (rounded as in the forward), sig = 1/(1+exp(-z)) and g the
 * gradient of out (rows, D) of dtype_g:
 *   d_y = g*s,  d_u = (g*s*d_skip)*coef,  d_z = (g*a)*sig*(1 + z*(1 - sig)),
 *   d_dskip = sum over rows of g*s*coef*u (deterministic)
 * in fp32, each rounded once to its input's element type; d_y, d_u, d_z are
 * (rows, D) contiguous, d_dskip (D,) float32.
 *   workspace >= m3_gate_bwd_workspace_bytes(rows, d_inner) bytes */
M3_API int m3_gate_bwd(int64_t rows, int32_t d_inner, const void* y, int32_t dtype_y,
            const void* u, int32_t dtype_u, const void* z, int32_t dtype_z, int64_t ld_z,
            const float* d_skip, float coef, int32_t round_silu, const void* g, int32_t dtype_g,
            void* d_y, void* d_u, void* d_z, float* d_dskip, void* workspace,
            size_t workspace_bytes, void* stream);

/* Size of the scratch buffer built into the library for m3_scan_bwd_noalloc. */
#define M3_NOALLOC_SCRATCH_BYTES (64u * 1024u * 1024u)

/* The analytic backward without a caller-supplied workspace.  No counterpart in
 * the reference: it exists for callers that cannot allocate device memory when
 * they run the backward (memory carved up at start-up by an allocator they have
 * no handle to, or loops that must not call cudaMalloc).  Inputs and outputs
 * are exactly those of m3_scan_bwd; the workspace comes from a device buffer of
 * M3_NOALLOC_SCRATCH_BYTES that the library holds on every GPU that loads it,
 * until the process exits.  This entry point never allocates or frees.
 *   - Problems whose m3_scan_bwd_workspace_bytes() exceeds the buffer are
 *     rejected with M3_ERR_SCRATCH_LIMIT.
 *   - The first call on each device looks up the buffer's device address (with
 *     that device current) and caches it; make that first call before any
 *     stream capture.  The cached address belongs to the device's current
 *     context: after cudaDeviceReset (or any other reset of the primary
 *     context) in the same process, this entry point must not be called
 *     again, since it would hand the kernels the stale address.
 *   - All calls on a device share the one buffer, which keeps the last call's
 *     contents.  Calls whose executions overlap on the GPU (other streams, or
 *     other host threads) race on it and corrupt each other's results. */
M3_API int m3_scan_bwd_noalloc(const m3_scan_desc* desc,
                const void* delta, const void* u, const void* Bc, const void* Cc,
                const float* A_real_p, const float* A_imag_p, const float* track_p,
                const void* dy, int32_t dtype_dy, const float* ckpt,
                void* d_delta, void* d_u, void* d_Bc, void* d_Cc,
                float* d_A_real_p, float* d_A_imag_p, float* d_track_p, void* stream);

/* ------------------------------------------------------------------------
 * Sequence-model operators beside the trapezoidal scan: layer and RMS norms
 * with their backward pass, the short causal convolution and the selective
 * scan (prompts, training, single tokens), and drawing a token from logits.
 * Row-strided inputs: row r starts at base + r * ld elements; a (B, L, .)
 * tensor has the rows b * L + t.  Arithmetic, states and sums are fp32 (64-bit
 * where stated); outputs are rounded once to their element type.  All results
 * are independent of scheduling (no floating-point atomics).  Batch, seqlen and
 * d_inner are at most 2^30 each; for the selective scan the products batch *
 * seqlen and batch * d_inner are below 2^31 and d_inner below 2^24. */

typedef struct m3_norm_desc {
  int64_t rows;       /* >= 1 */
  int32_t d;          /* 1..32768 */
  int32_t dtype_x;    /* element type of x and dx */
  int32_t dtype_y;    /* element type of y and g */
  int32_t rms;        /* non-zero: RMS norm (no mean, no bias) */
  float eps;          /* >= 0 */
} m3_norm_desc;

/* y = (x - mean) * rstd * w + b over rows of d elements, rstd =
 * 1 / sqrt(mean((x - mean)^2) + eps); mean is 0 for the RMS norm (the RMSNorm
 * of mamba.py:82-89; the layer norms of search_mamba.py's heads).
 *   x (rows, ld_x); w (d,) float32; b (d,) float32 or NULL (NULL for the RMS norm);
 *   y (rows, d)
 *   mean, rstd (rows,) float32 for the backward, or NULL.  y may be x when
 *   ld_x == d and both have one element type. */
M3_API int m3_norm_fwd(const m3_norm_desc* desc, const void* x, int64_t ld_x, const float* w,
            const float* b, void* y, float* mean, float* rstd, void* stream);

/* Workspace bytes of m3_norm_bwd on the current device. */
M3_API size_t m3_norm_bwd_workspace_bytes(const m3_norm_desc* desc);

/* Backward of m3_norm_fwd: g (rows, d) the gradient of y; dx (rows, d); dw and
 * db (d,) float32 (db NULL when there is no bias); mean is not read for the RMS
 * norm.  The weight gradients are summed over the rows in a fixed order. */
M3_API int m3_norm_bwd(const m3_norm_desc* desc, const void* x, int64_t ld_x, const float* w,
            const float* mean, const float* rstd, const void* g, void* dx, float* dw, float* db,
            void* workspace, size_t workspace_bytes, void* stream);

typedef struct m3_add_norm_desc {
  int64_t rows;       /* >= 1 */
  int32_t d;          /* 1..32768 */
  int32_t dtype_x;    /* element type of the branch x and of dx */
  int32_t dtype_s;    /* element type of the residual stream: res, s, gs, ds */
  int32_t dtype_y;    /* element type of y and gy */
  float eps;          /* >= 0 */
} m3_add_norm_desc;

/* The residual's addition and the RMS norm behind it (mamba.py:591-595 and 82-89):
 *   s = x + res, rounded to dtype_s;  y = s * rstd * w, rstd = 1 / sqrt(mean(s^2) + eps)
 *   x (rows, ld_x), res (rows, ld_r), w (d,) float32, y and s (rows, d), rstd
 *   (rows,) float32 for the backward, or NULL.  s may be res when ld_r == d, or x
 *   when ld_x == d and both have one element type; no other output shares bytes
 *   with an input or another output (M3_ERR_ALIAS). */
M3_API int m3_add_norm_fwd(const m3_add_norm_desc* desc, const void* x, int64_t ld_x,
            const void* res, int64_t ld_r, const float* w, void* y, void* s, float* rstd,
            void* stream);

/* Backward: s (rows, ld_s) and rstd of the forward, gy (rows, d) the gradient of
 * y, gs (rows, d) that of s or NULL (zero).  ds (rows, d) is the gradient of res;
 * dx (rows, d) that of x where dtype_x is not dtype_s, else NULL (ds serves).  dw
 * (d,) float32, summed over the rows in a fixed order.  ds may be gs; no other
 * output shares bytes with an input or another output (M3_ERR_ALIAS). */
M3_API size_t m3_add_norm_bwd_workspace_bytes(const m3_add_norm_desc* desc);
M3_API int m3_add_norm_bwd(const m3_add_norm_desc* desc, const void* s, int64_t ld_s,
            const float* w, const float* rstd, const void* gy, const void* gs, void* ds, void* dx,
            float* dw, void* workspace, size_t workspace_bytes, void* stream);

typedef struct m3_norm8_desc {
  int64_t rows;       /* >= 1 */
  int32_t d;          /* 1..32768 */
  int32_t group;      /* columns per scale: 32, 64 or 128 that divide d, or 0: a row */
  int32_t dtype_x;    /* element type of x */
  int32_t dtype_s;    /* element type of res and s */
  int32_t e4m3;       /* non-zero: 8-bit floats (largest value 448), else int8 (127) */
  float eps;          /* >= 0 */
} m3_norm8_desc;

/* y = the RMS norm of x, or of s = x + res rounded to dtype_s, in 8 bits:
 *   scale = max(max |y| / top, 2^-126) over a row or a group of columns, to 2^-23 of it,
 *   q = y / scale, formed to 2^-22 of itself, then rounded to nearest even and held to
 *   [-top, top] (a quotient that near to the border of two codes may get either)
 *   x (rows, ld_x), res (rows, ld_r) or NULL, w (d,) float32, q (rows, d) bytes,
 *   scale (rows,) or (rows, d / group) float32, s (rows, d), not used without res.
 * A group with a NaN has the scale NaN.  With groups, rows and pointers aligned to
 * 4 elements (q to 4 bytes).  s may be res or x, as in m3_add_norm_fwd; no other
 * output shares bytes with an input or another output (M3_ERR_ALIAS). */
M3_API int m3_norm8_fwd(const m3_norm8_desc* desc, const void* x, int64_t ld_x, const void* res,
            int64_t ld_r, const float* w, void* q, float* scale, void* s, void* stream);

typedef struct m3_conv_desc {
  int32_t batch;      /* B >= 1 */
  int32_t seqlen;     /* L >= 1; 1 for the step */
  int32_t d_inner;    /* D >= 1 */
  int32_t width;      /* K taps, 1..8 */
  int32_t dtype;      /* element type of x, y, the state and their gradients */
  int32_t silu;       /* non-zero: y = silu(p), else y = p */
} m3_conv_desc;

/* Causal convolution over time, one filter per channel:
 *   p[b,t,d] = bias[d] + sum_k w[d,k] x[b, t-K+1+k, d]
 *   x (B*L, ld_x); w (D, K) float32; b (D,) float32 or NULL; y (B, L, D)
 *   state      (B, K-1, D) or NULL (zeros): the input rows before x, oldest first
 *   lengths    (B,) int32 or NULL (all L), clamped to [0, L]: steps at or past a
 *              row's length are not read, and y is zero there
 *   state_out  (B, K-1, D) or NULL: the last K-1 rows of [state; x[:length]];
 *              must not be state, nor y x. */
M3_API int m3_causal_conv_fwd(const m3_conv_desc* desc, const void* x, int64_t ld_x,
            const float* w, const float* b, const void* state, const int32_t* lengths, void* y,
            void* state_out, void* stream);

/* Workspace bytes of m3_causal_conv_bwd on the current device. */
M3_API size_t m3_causal_conv_bwd_workspace_bytes(const m3_conv_desc* desc);

/* Backward: g (B, L, D) the gradient of y; dx (B, L, D), zero at steps past a
 * length; dw (D, K), db (D,) float32 (db may be NULL without a bias).  The state
 * gets no gradient.  dx must be neither x nor g. */
M3_API int m3_causal_conv_bwd(const m3_conv_desc* desc, const void* x, int64_t ld_x,
            const float* w, const float* b, const void* state, const int32_t* lengths,
            const void* g, void* dx, float* dw, float* db, void* workspace,
            size_t workspace_bytes, void* stream);

/* One token per row (seqlen 1): y (B, D) from [state; x], x (B, ld_x); the
 * state (B, K-1, D) moves up by one row in place. */
M3_API int m3_causal_conv_step(const m3_conv_desc* desc, void* state, const void* x, int64_t ld_x,
            const float* w, const float* b, void* y, void* stream);

typedef struct m3_sel_desc {
  int32_t batch;      /* B >= 1 */
  int32_t seqlen;     /* L >= 1; 1 for the step */
  int32_t d_inner;    /* D >= 1 */
  int32_t d_state;    /* N, 1..128 */
  int32_t dtype;      /* element type of u, dt, z, B, C, y and their gradients */
  int32_t softplus;   /* non-zero: step size softplus(dt + dt_bias), else dt + dt_bias */
} m3_sel_desc;

typedef struct m3_sel_args {
  const void* u;  int64_t ld_u;     /* (B*L, ld_u), D columns */
  const void* dt; int64_t ld_dt;    /* (B*L, ld_dt), D columns */
  const void* z;  int64_t ld_z;     /* (B*L, ld_z), D columns, or NULL: no gate */
  const void* B;  int64_t ld_b;     /* (B*L, ld_b), N columns */
  const void* C;  int64_t ld_c;     /* (B*L, ld_c), N columns */
  const float* A;                   /* (D, N) */
  const float* d_skip;              /* (D,) or NULL */
  const float* dt_bias;             /* (D,) or NULL */
  const float* state;               /* (B, D, N) the state before the first step, or NULL: zero */
  const int32_t* lengths;           /* (B,) or NULL: all L; clamped to [0, L] */
} m3_sel_args;

/* Selective scan, per row b, channel d and state n:
 *   de_t = softplus(dt_t + dt_bias),   h_t = exp(de_t A) h_{t-1} + de_t u_t B_t
 *   y_t  = (sum_n C_t h_t + d_skip u_t) * silu(z_t)
 *   y       (B, L, D); zero at steps at or past a row's length, whose inputs are
 *           not read
 *   h_last  (B, D, N) float32 or NULL: the state at each row's length (not state)
 *   ckpt    m3_selective_ckpt_floats() floats for the backward, 16-byte aligned,
 *           or NULL
 *   workspace >= m3_selective_fwd_workspace_bytes() bytes (0 for large batches;
 *           few rows are split along time), 16-byte aligned */
M3_API size_t m3_selective_ckpt_floats(const m3_sel_desc* desc);
M3_API size_t m3_selective_fwd_workspace_bytes(const m3_sel_desc* desc);
M3_API int m3_selective_fwd(const m3_sel_desc* desc, const m3_sel_args* args, void* y,
            float* h_last, float* ckpt, void* workspace, size_t workspace_bytes, void* stream);

typedef struct m3_sel_grads {
  void* d_u; void* d_dt; void* d_z;          /* (B, L, D); d_z unused without z */
  void* d_B; void* d_C;                      /* (B, L, N), aligned to 4 elements */
  float* d_A;                                /* (D, N) */
  float* d_skip; float* d_dt_bias;           /* (D,) or NULL */
} m3_sel_grads;

/* Backward of m3_selective_fwd: g (B, L, D) the gradient of y, ckpt the
 * forward's.  The states get no gradient.  The batch is taken in slabs of rows
 * whose partials of d_B and d_C (0.5, 2, 8, 16, 64 bytes per step and channel for
 * up to 8, 16, 32, 64, 128 states) fill 2 GB, or in larger ones of the rows that
 * one wave of CTAs walks. */
M3_API size_t m3_selective_bwd_workspace_bytes(const m3_sel_desc* desc);
M3_API int m3_selective_bwd(const m3_sel_desc* desc, const m3_sel_args* args, const void* g,
            const float* ckpt, const m3_sel_grads* grads, void* workspace,
            size_t workspace_bytes, void* stream);

/* One token per row (seqlen 1), in place on h (B, D, N) float32; y (B, D).
 * args->state and args->lengths must be NULL; at most 524280 rows. */
M3_API int m3_selective_step(const m3_sel_desc* desc, const m3_sel_args* args, float* h, void* y,
            void* stream);

typedef struct m3_gated_desc {
  int32_t batch;      /* B >= 1 */
  int32_t seqlen;     /* L >= 1; 1 for the step */
  int32_t d_inner;    /* D >= 1 */
  int32_t dtype;      /* element type of x, rg, ig, y and their gradients */
  float c;            /* > 0, finite */
} m3_gated_desc;

typedef struct m3_gated_args {
  const void* x;  int64_t ld_x;     /* (B*L, ld_x), D columns: the input */
  const void* rg; int64_t ld_r;     /* (B*L, ld_r): recurrence gate before its sigmoid */
  const void* ig; int64_t ld_i;     /* (B*L, ld_i): input gate before its sigmoid */
  const float* decay;               /* (D,) */
  const float* state;               /* (B, D) the state before the first step, or NULL: zero */
  const int32_t* lengths;           /* (B,) or NULL: all L; clamped to [0, L] */
} m3_gated_args;

/* Gated linear recurrence, per row b and channel d:
 *   a_t = exp(-c softplus(decay) sigmoid(rg_t)),
 *   h_t = a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(ig_t) x_t,   y_t = h_t
 *   y       (B, L, D); zero at steps at or past a row's length, whose inputs are
 *           not read
 *   h_last  (B, D) float32 or NULL: the state at each row's length (not state)
 *   ckpt    m3_gated_ckpt_floats() floats for the backward (the state in front of
 *           every 4 steps), 8-byte aligned, or NULL
 * Here and below an output that shares bytes with an input or another output is
 * refused (M3_ERR_ALIAS). */
M3_API size_t m3_gated_ckpt_floats(const m3_gated_desc* desc);
M3_API int m3_gated_fwd(const m3_gated_desc* desc, const m3_gated_args* args, void* y,
            float* h_last, float* ckpt, void* stream);

/* Backward: g (B, L, D) the gradient of y, ckpt the forward's; d_x, d_rg, d_ig
 * (B, L, D), zero at steps at or past a length; d_decay (D,) float32, summed in a
 * fixed order.  The states get no gradient. */
M3_API size_t m3_gated_bwd_workspace_bytes(const m3_gated_desc* desc);
M3_API int m3_gated_bwd(const m3_gated_desc* desc, const m3_gated_args* args, const void* g,
            const float* ckpt, void* d_x, void* d_rg, void* d_ig, float* d_decay,
            void* workspace, size_t workspace_bytes, void* stream);

/* One token per row (seqlen 1), in place on h (B, D) float32; y (B, D).
 * args->state and args->lengths must be NULL. */
M3_API int m3_gated_step(const m3_gated_desc* desc, const m3_gated_args* args, float* h, void* y,
            void* stream);

typedef struct m3_sample_desc {
  int32_t rows;         /* >= 1 */
  int32_t vocab;        /* V, 1..262144 */
  int32_t dtype;        /* element type of logits */
  float temperature;    /* settings of every row, where no array is given */
  int32_t top_k;
  float top_p;
  float min_p;
} m3_sample_desc;

/* Draws one token per row.  With w_i = exp((x_i - max) / temperature) over the
 * candidates (x_i neither -infinity nor NaN; where the maximum is +infinity its
 * holders weigh 1 and the others 0), ordered by x descending, then index:
 *   top_k   keeps the first k (<= 0: all)
 *   top_p   of those, the shortest prefix with at least top_p of their weight,
 *           one token at least (>= 1: all; negative or NaN: as 0, one token)
 *   min_p   of those, the tokens with w_i >= min(min_p, 1)
 * and the token is the smallest index whose cumulative weight over the kept
 * tokens, in index order, exceeds uniform * their total (the last kept one when
 * none does).  temperature <= 0 or NaN takes the first token of the order; a row
 * without candidates gives -1.  Weights are summed as 64-bit integers of the
 * double-precision exponentials.
 *   logits (rows, ld); uniform (rows,) in [0, 1); temperature, top_p, min_p
 *   (rows,) float32 and top_k (rows,) int32 arrays override the descriptor's
 *   values where not NULL; out (rows,) int64. */
M3_API int m3_sample(const m3_sample_desc* desc, const void* logits, int64_t ld,
            const float* uniform, const float* temperature, const int32_t* top_k,
            const float* top_p, const float* min_p, int64_t* out, void* stream);

/* Reads (and clears when clear != 0) the device-side error word of the
 * current device; *code receives 0 or an M3_ERR_* value. */
M3_API int m3_device_error(int32_t* code, int32_t clear);

#ifdef __cplusplus
}
#endif

#endif /* M3SCAN_H */
