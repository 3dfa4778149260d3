// C ABI of the sequence-model operators: argument validation, plans, workspace
// layout and dispatch.  No allocation, no exceptions, no host sync.
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include "m3_api_util.h"
#include "m3_ops.h"
#include "m3scan.h"

using namespace m3;

namespace {

int status(cudaError_t e) {
  if (e == cudaSuccess) return M3_OK;
  cudaGetLastError();
  return M3_ERR_LAUNCH;
}

// sizes that the kernels' 32-bit roundings up to tiles could pass 2^31 with
bool too_large(int a, int b, int c) {
  constexpr int most = 1 << 30;
  return a > most || b > most || c > most;
}

int check_norm(const m3_norm_desc* d) {
  if (!d) return M3_ERR_NULL;
  if (d->rows < 1 || d->d < 1 || !(d->eps >= 0.f)) return M3_ERR_SHAPE;
  if (!dtype_ok(d->dtype_x) || !dtype_ok(d->dtype_y)) return M3_ERR_DTYPE;
  if (d->d > kMaxNormD) return M3_ERR_UNSUPPORTED;
  return M3_OK;
}

int check_conv(const m3_conv_desc* d) {
  if (!d) return M3_ERR_NULL;
  if (d->batch < 1 || d->seqlen < 1 || d->d_inner < 1 || d->width < 1) return M3_ERR_SHAPE;
  if (too_large(d->batch, d->seqlen, d->d_inner)) return M3_ERR_SHAPE;
  if ((double)d->batch * d->seqlen * d->d_inner > 128.0 * 2147483647.0) return M3_ERR_SHAPE;
  if (!dtype_ok(d->dtype)) return M3_ERR_DTYPE;
  if (d->width > kMaxConvWidth) return M3_ERR_UNSUPPORTED;
  return M3_OK;
}

int check_sel(const m3_sel_desc* d) {
  if (!d) return M3_ERR_NULL;
  if (d->batch < 1 || d->seqlen < 1 || d->d_inner < 1 || d->d_state < 1) return M3_ERR_SHAPE;
  if (!dtype_ok(d->dtype)) return M3_ERR_DTYPE;
  if (d->d_state > kMaxSelState) return M3_ERR_UNSUPPORTED;
  if (too_large(d->batch, d->seqlen, d->d_inner)) return M3_ERR_SHAPE;
  // grids: rows x channel tiles, state quads of the joins
  const double tiles = (double)(d->d_inner + 15) / 16;
  if (tiles > 65535.0 * 16 || (double)d->batch * tiles > 2147483647.0 ||
      (double)d->batch * d->seqlen > 2147483647.0 ||
      (double)d->batch * d->d_inner > 2147483647.0)
    return M3_ERR_SHAPE;
  return M3_OK;
}

// Few rows are split along time into runs, of four chunks at least.  The
// summaries of the runs cost about three quarters of another pass, so fewer
// than three runs do not pay.
int time_splits(int nch, long long ctas, long long want) {
  long long s = want / ctas;
  if (s > nch / 4) s = nch / 4;
  if (s < 3) return 1;
  const int cps = (int)((nch + s - 1) / s);
  return (nch + cps - 1) / cps;
}

// The backward's partials of dB and dC: rows are taken in slabs of this many
// bytes, or of the rows that one wave of CTAs walks where those need more.
constexpr size_t kSelSlabBytes = (size_t)2 << 30;

struct SelLayout {
  int splits, cps, nch, np, tiles, bgroups, workers;
  int slab;                            // rows of the batch that the backward takes at a time
  size_t hin, hsum, dsum;              // the time split's buffers (backward: qin, qsum)
  size_t bc, a;                        // the backward's partials
  size_t total;
};

bool sel_layout(const m3_sel_desc* d, bool backward, SelLayout* l) {
  const int sms = device_sms();
  if (sms <= 0) return false;
  const int per = backward ? sel_bwd_resident(d->d_state, d->dtype)
                           : sel_fwd_resident(d->d_state, d->dtype);
  if (per <= 0) return false;
  const int ln = sel_lanes(d->d_state);
  const int tile = backward ? sel_tile(ln) : sel_fwd_tile(d->d_state);
  const long long wave = (long long)per * sms;
  l->np = 4 * ln;
  l->nch = (d->seqlen + kSelSteps - 1) / kSelSteps;
  l->tiles = (d->d_inner + tile - 1) / tile;
  // runs for two waves forward and three backward, whose summaries run on
  // narrower CTAs than the pass itself (2 x 4001 x 1536 steps, N = 16, fp32:
  // 544 us against 608 us for one and two waves)
  l->splits = time_splits(l->nch, (long long)d->batch * l->tiles, (backward ? 3 : 2) * wave);
  l->cps = (l->nch + l->splits - 1) / l->splits;
  // backward: CTAs walk rows of the batch, one wave of them
  long long bg = wave / ((long long)l->tiles * l->splits);
  if (bg > d->batch) bg = d->batch;
  if (bg < 1) bg = 1;
  const size_t row_bc = (size_t)l->tiles * d->seqlen * 2 * l->np * 4;
  long long slab = (long long)(kSelSlabBytes / row_bc);
  if (slab < bg) slab = bg;
  if (slab > d->batch) slab = d->batch;
  const long long slabs = (d->batch + slab - 1) / slab;
  l->slab = (int)((d->batch + slabs - 1) / slabs);   // of equal size
  if (bg > l->slab) bg = l->slab;
  l->bgroups = (int)bg;
  l->workers = l->bgroups * l->splits;
  const size_t run = round256((size_t)l->splits * d->batch * d->d_inner * l->np * 4);
  const size_t sums = round256((size_t)l->splits * d->batch * d->d_inner * 4);
  l->hin = 0;
  l->hsum = run;
  l->dsum = 2 * run;
  l->bc = l->splits > 1 ? 2 * run + sums : 0;
  l->total = l->bc;
  if (backward) {
    l->a = l->bc + round256(l->slab * row_bc);
    l->total = l->a + round256((size_t)l->workers * d->d_inner * (l->np + 2) * 4);
  }
  return true;
}

// Fills what forward and backward share; returns a status.
int fill_sel(const m3_sel_desc* d, const m3_sel_args* a, const SelLayout& l, SelParams* p) {
  const int e = dsize(d->dtype);
  if (!a) return M3_ERR_NULL;
  if (!a->u || !a->dt || !a->A || !a->B || !a->C) return M3_ERR_NULL;
  if (a->ld_u < d->d_inner || a->ld_dt < d->d_inner || (a->z && a->ld_z < d->d_inner) ||
      a->ld_b < d->d_state || a->ld_c < d->d_state)
    return M3_ERR_SHAPE;
  if (!aligned(a->u, e) || !aligned(a->dt, e) || !aligned(a->z, e) || !aligned(a->B, e) ||
      !aligned(a->C, e) || !aligned(a->A, 4) || !aligned(a->d_skip, 4) ||
      !aligned(a->dt_bias, 4) || !aligned(a->state, 4) || !aligned(a->lengths, 4))
    return M3_ERR_ALIGN;
  p->u = a->u; p->dt = a->dt; p->z = a->z; p->Bm = a->B; p->Cm = a->C;
  p->ld_u = a->ld_u; p->ld_dt = a->ld_dt; p->ld_z = a->ld_z; p->ld_b = a->ld_b;
  p->ld_c = a->ld_c;
  p->A = a->A; p->dskip = a->d_skip; p->dt_bias = a->dt_bias; p->h0 = a->state;
  p->lengths = a->lengths;
  p->B = d->batch; p->L = d->seqlen; p->D = d->d_inner; p->N = d->d_state;
  p->dtype = d->dtype; p->softplus = d->softplus != 0;
  p->nch = l.nch; p->splits = l.splits; p->cps = l.cps;
  const int v = 16 / e;   // elements of the widest load
  p->vec_d = d->d_inner % v == 0 && a->ld_u % v == 0 && a->ld_dt % v == 0 &&
             (!a->z || a->ld_z % v == 0) && aligned(a->u, 16) && aligned(a->dt, 16) &&
             aligned(a->z, 16);
  p->vec_n = d->d_state % 4 == 0 && a->ld_b % 4 == 0 && a->ld_c % 4 == 0 &&
             aligned(a->B, 4 * e) && aligned(a->C, 4 * e);
  return M3_OK;
}

}  // namespace

extern "C" {

int m3_norm_fwd(const m3_norm_desc* desc, const void* x, int64_t ld_x, const float* w,
                const float* b, void* y, float* mean, float* rstd, void* stream) {
  int rc = check_norm(desc);
  if (rc != M3_OK) return rc;
  if (ld_x < desc->d) return M3_ERR_SHAPE;
  if (!x || !w || !y) return M3_ERR_NULL;
  if (desc->rms && b) return M3_ERR_UNSUPPORTED;   // it has no bias
  if (!aligned(x, dsize(desc->dtype_x)) || !aligned(y, dsize(desc->dtype_y)) ||
      !aligned(w, 4) || !aligned(b, 4) || !aligned(mean, 4) || !aligned(rstd, 4))
    return M3_ERR_ALIGN;
  if ((rc = check_device()) != M3_OK) return rc;
  NormParams p;
  memset(&p, 0, sizeof(p));
  p.x = x; p.ld_x = ld_x; p.w = w; p.b = b; p.y = y; p.mean = mean; p.rstd = rstd;
  p.rows = desc->rows; p.d = desc->d;
  p.dtype_x = desc->dtype_x; p.dtype_y = desc->dtype_y; p.rms = desc->rms != 0;
  p.eps = desc->eps;
  p.sms = device_sms();
  return status(launch_norm_fwd(p, static_cast<cudaStream_t>(stream)));
}

size_t m3_norm_bwd_workspace_bytes(const m3_norm_desc* desc) {
  const int sms = device_sms();
  if (check_norm(desc) != M3_OK || sms <= 0) return 0;
  return (size_t)norm_bwd_ctas(desc->rows, desc->d, sms) * 2 * desc->d * 4;
}

int m3_norm_bwd(const m3_norm_desc* desc, const void* x, int64_t ld_x, const float* w,
                const float* mean, const float* rstd, const void* g, void* dx, float* dw,
                float* db, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_norm(desc);
  if (rc != M3_OK) return rc;
  if (ld_x < desc->d) return M3_ERR_SHAPE;
  if (!x || !w || !rstd || (!desc->rms && !mean) || !g || !dx || !dw) return M3_ERR_NULL;
  if (desc->rms && db) return M3_ERR_UNSUPPORTED;   // it has no bias
  if (!aligned(x, dsize(desc->dtype_x)) || !aligned(dx, dsize(desc->dtype_x)) ||
      !aligned(g, dsize(desc->dtype_y)) || !aligned(w, 4) || !aligned(mean, 4) ||
      !aligned(rstd, 4) || !aligned(dw, 4) || !aligned(db, 4) || !aligned(workspace, 4))
    return M3_ERR_ALIGN;
  if ((rc = check_device()) != M3_OK) return rc;
  if (!workspace || workspace_bytes < m3_norm_bwd_workspace_bytes(desc)) return M3_ERR_WORKSPACE;
  NormBwdParams p;
  memset(&p, 0, sizeof(p));
  p.x = x; p.ld_x = ld_x; p.w = w; p.mean = mean; p.rstd = rstd; p.g = g; p.dx = dx;
  p.dw = dw; p.db = db; p.part = static_cast<float*>(workspace);
  p.rows = desc->rows; p.d = desc->d;
  p.dtype_x = desc->dtype_x; p.dtype_y = desc->dtype_y; p.rms = desc->rms != 0;
  p.sms = device_sms();
  return status(launch_norm_bwd(p, static_cast<cudaStream_t>(stream)));
}

int m3_causal_conv_fwd(const m3_conv_desc* desc, const void* x, int64_t ld_x, const float* w,
                       const float* b, const void* state, const int32_t* lengths, void* y,
                       void* state_out, void* stream) {
  int rc = check_conv(desc);
  if (rc != M3_OK) return rc;
  if (ld_x < desc->d_inner) return M3_ERR_SHAPE;
  if (!x || !w || !y) return M3_ERR_NULL;
  const int e = dsize(desc->dtype);
  if (!aligned(x, e) || !aligned(y, e) || !aligned(state, e) || !aligned(state_out, e) ||
      !aligned(w, 4) || !aligned(b, 4) || !aligned(lengths, 4))
    return M3_ERR_ALIGN;
  if (y == x || (state_out && state_out == state)) return M3_ERR_ALIAS;
  if ((rc = check_device()) != M3_OK) return rc;
  ConvParams p;
  memset(&p, 0, sizeof(p));
  p.x = x; p.ld_x = ld_x; p.w = w; p.b = b; p.state = state; p.lengths = lengths; p.y = y;
  p.state_out = state_out;
  p.B = desc->batch; p.L = desc->seqlen; p.D = desc->d_inner; p.K = desc->width;
  p.dtype = desc->dtype; p.silu = desc->silu != 0;
  p.sms = device_sms();
  return status(launch_conv_fwd(p, static_cast<cudaStream_t>(stream)));
}

size_t m3_causal_conv_bwd_workspace_bytes(const m3_conv_desc* desc) {
  const int sms = device_sms();
  if (check_conv(desc) != M3_OK || sms <= 0) return 0;
  int workers, tt;
  conv_bwd_plan(desc->batch, desc->seqlen, desc->d_inner, sms, &workers, &tt);
  return (size_t)workers * (desc->width + 1) * desc->d_inner * 4;
}

int m3_causal_conv_bwd(const m3_conv_desc* desc, const void* x, int64_t ld_x, const float* w,
                       const float* b, const void* state, const int32_t* lengths, const void* g,
                       void* dx, float* dw, float* db, void* workspace, size_t workspace_bytes,
                       void* stream) {
  int rc = check_conv(desc);
  if (rc != M3_OK) return rc;
  if (ld_x < desc->d_inner) return M3_ERR_SHAPE;
  if (!x || !w || !g || !dx || !dw || (b && !db)) return M3_ERR_NULL;
  const int e = dsize(desc->dtype);
  if (!aligned(x, e) || !aligned(g, e) || !aligned(dx, e) || !aligned(state, e) ||
      !aligned(w, 4) || !aligned(b, 4) || !aligned(lengths, 4) || !aligned(dw, 4) ||
      !aligned(db, 4) || !aligned(workspace, 4))
    return M3_ERR_ALIGN;
  if (dx == x || dx == g) return M3_ERR_ALIAS;
  if ((rc = check_device()) != M3_OK) return rc;
  if (!workspace || workspace_bytes < m3_causal_conv_bwd_workspace_bytes(desc))
    return M3_ERR_WORKSPACE;
  ConvBwdParams p;
  memset(&p, 0, sizeof(p));
  p.x = x; p.ld_x = ld_x; p.w = w; p.b = b; p.state = state; p.lengths = lengths; p.g = g;
  p.dx = dx; p.dw = dw; p.db = db; p.part = static_cast<float*>(workspace);
  p.B = desc->batch; p.L = desc->seqlen; p.D = desc->d_inner; p.K = desc->width;
  p.dtype = desc->dtype; p.silu = desc->silu != 0;
  p.sms = device_sms();
  conv_bwd_plan(p.B, p.L, p.D, p.sms, &p.workers, &p.tt);
  return status(launch_conv_bwd(p, static_cast<cudaStream_t>(stream)));
}

int m3_causal_conv_step(const m3_conv_desc* desc, void* state, const void* x, int64_t ld_x,
                        const float* w, const float* b, void* y, void* stream) {
  int rc = check_conv(desc);
  if (rc != M3_OK) return rc;
  if (ld_x < desc->d_inner || desc->seqlen != 1) return M3_ERR_SHAPE;
  if (!x || !w || !y || (desc->width > 1 && !state)) return M3_ERR_NULL;
  const int e = dsize(desc->dtype);
  if (!aligned(x, e) || !aligned(y, e) || !aligned(state, e) || !aligned(w, 4) || !aligned(b, 4))
    return M3_ERR_ALIGN;
  if (y == state || x == state) return M3_ERR_ALIAS;
  if ((rc = check_device()) != M3_OK) return rc;
  ConvStepParams p;
  memset(&p, 0, sizeof(p));
  p.state = state; p.x = x; p.ld_x = ld_x; p.w = w; p.b = b; p.y = y;
  p.B = desc->batch; p.D = desc->d_inner; p.K = desc->width;
  p.dtype = desc->dtype; p.silu = desc->silu != 0;
  return status(launch_conv_step(p, static_cast<cudaStream_t>(stream)));
}

size_t m3_selective_ckpt_floats(const m3_sel_desc* desc) {
  if (check_sel(desc) != M3_OK) return 0;
  const int nch = (desc->seqlen + kSelSteps - 1) / kSelSteps;
  return (size_t)desc->batch * (nch - 1) * desc->d_inner * 4 * sel_lanes(desc->d_state);
}

size_t m3_selective_fwd_workspace_bytes(const m3_sel_desc* desc) {
  SelLayout l;
  if (check_sel(desc) != M3_OK || !sel_layout(desc, false, &l)) return 0;
  return l.total;
}

int m3_selective_fwd(const m3_sel_desc* desc, const m3_sel_args* args, void* y, float* h_last,
                     float* ckpt, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_sel(desc);
  if (rc != M3_OK) return rc;
  if (!args || !y) return M3_ERR_NULL;
  if (!aligned(y, dsize(desc->dtype)) || !aligned(h_last, 4) || !aligned(ckpt, 16) ||
      !aligned(workspace, 16))
    return M3_ERR_ALIGN;
  if (h_last && h_last == args->state) return M3_ERR_ALIAS;
  SelParams p;
  memset(&p, 0, sizeof(p));
  SelLayout l;
  memset(&l, 0, sizeof(l));
  if ((rc = fill_sel(desc, args, l, &p)) != M3_OK) return rc;
  if ((rc = check_device()) != M3_OK) return rc;
  if (!sel_layout(desc, false, &l)) return M3_ERR_NO_DEVICE;
  if (l.total && (!workspace || workspace_bytes < l.total)) return M3_ERR_WORKSPACE;
  fill_sel(desc, args, l, &p);
  p.vec_d = p.vec_d && aligned(y, 16);
  p.y = y; p.h_last = h_last; p.ckpt = l.nch > 1 ? ckpt : nullptr;
  if (l.splits > 1) {
    char* ws = static_cast<char*>(workspace);
    p.hin = reinterpret_cast<float*>(ws + l.hin);
    p.hsum = reinterpret_cast<float*>(ws + l.hsum);
    p.dsum = reinterpret_cast<float*>(ws + l.dsum);
  }
  return status(launch_sel_fwd(p, static_cast<cudaStream_t>(stream)));
}

size_t m3_selective_bwd_workspace_bytes(const m3_sel_desc* desc) {
  SelLayout l;
  if (check_sel(desc) != M3_OK || !sel_layout(desc, true, &l)) return 0;
  return l.total;
}

int m3_selective_bwd(const m3_sel_desc* desc, const m3_sel_args* args, const void* g,
                     const float* ckpt, const m3_sel_grads* grads, void* workspace,
                     size_t workspace_bytes, void* stream) {
  int rc = check_sel(desc);
  if (rc != M3_OK) return rc;
  if (!args || !g || !grads) return M3_ERR_NULL;
  if (!grads->d_u || !grads->d_dt || (args->z && !grads->d_z) || !grads->d_A || !grads->d_B ||
      !grads->d_C)
    return M3_ERR_NULL;
  const int e = dsize(desc->dtype);
  if (!aligned(g, e) || !aligned(grads->d_u, e) || !aligned(grads->d_dt, e) ||
      !aligned(grads->d_z, e) || !aligned(grads->d_B, 4 * e) || !aligned(grads->d_C, 4 * e) ||
      !aligned(grads->d_A, 4) || !aligned(grads->d_skip, 4) || !aligned(grads->d_dt_bias, 4) ||
      !aligned(ckpt, 16) || !aligned(workspace, 16))
    return M3_ERR_ALIGN;
  SelBwdParams p;
  memset(&p, 0, sizeof(p));
  SelLayout l;
  memset(&l, 0, sizeof(l));
  if ((rc = fill_sel(desc, args, l, &p.f)) != M3_OK) return rc;
  if ((rc = check_device()) != M3_OK) return rc;
  if (!sel_layout(desc, true, &l)) return M3_ERR_NO_DEVICE;
  if (!workspace || workspace_bytes < l.total) return M3_ERR_WORKSPACE;
  if (l.nch > 1 && !ckpt) return M3_ERR_NULL;
  fill_sel(desc, args, l, &p.f);
  p.f.ckpt = const_cast<float*>(ckpt);
  p.g = g;
  p.du = grads->d_u; p.ddt = grads->d_dt; p.dz = grads->d_z; p.dB = grads->d_B;
  p.dC = grads->d_C; p.dA = grads->d_A; p.dD = grads->d_skip; p.dbias = grads->d_dt_bias;
  char* ws = static_cast<char*>(workspace);
  p.part_bc = reinterpret_cast<float*>(ws + l.bc);
  p.part_a = reinterpret_cast<float*>(ws + l.a);
  if (l.splits > 1) {
    p.qin = reinterpret_cast<float*>(ws + l.hin);
    p.qsum = reinterpret_cast<float*>(ws + l.hsum);
    p.f.dsum = reinterpret_cast<float*>(ws + l.dsum);
  }
  p.workers = l.workers;
  p.bgroups = l.bgroups;
  p.nb = l.slab;
  p.vec_g = desc->d_inner % (16 / e) == 0 && aligned(g, 16) && aligned(grads->d_u, 16) &&
            aligned(grads->d_dt, 16) && aligned(grads->d_z, 16);
  return status(launch_sel_bwd(p, static_cast<cudaStream_t>(stream)));
}

int m3_selective_step(const m3_sel_desc* desc, const m3_sel_args* args, float* h, void* y,
                      void* stream) {
  int rc = check_sel(desc);
  if (rc != M3_OK) return rc;
  if (desc->seqlen != 1 || desc->batch > 65535 * 8) return M3_ERR_SHAPE;
  if (!args || !h || !y) return M3_ERR_NULL;
  if (!aligned(h, 4) || !aligned(y, dsize(desc->dtype))) return M3_ERR_ALIGN;
  if (args->state || args->lengths) return M3_ERR_UNSUPPORTED;   // the state is h
  SelParams f;
  memset(&f, 0, sizeof(f));
  SelLayout l;
  memset(&l, 0, sizeof(l));
  if ((rc = fill_sel(desc, args, l, &f)) != M3_OK) return rc;
  if ((rc = check_device()) != M3_OK) return rc;
  SelStepParams p;
  memset(&p, 0, sizeof(p));
  p.h = h; p.u = f.u; p.dt = f.dt; p.z = f.z; p.Bm = f.Bm; p.Cm = f.Cm;
  p.ld_u = f.ld_u; p.ld_dt = f.ld_dt; p.ld_z = f.ld_z; p.ld_b = f.ld_b; p.ld_c = f.ld_c;
  p.A = f.A; p.dskip = f.dskip; p.dt_bias = f.dt_bias; p.y = y;
  p.B = f.B; p.D = f.D; p.N = f.N; p.dtype = f.dtype; p.softplus = f.softplus;
  return status(launch_sel_step(p, static_cast<cudaStream_t>(stream)));
}

int m3_sample(const m3_sample_desc* desc, const void* logits, int64_t ld, const float* uniform,
              const float* temperature, const int32_t* top_k, const float* top_p,
              const float* min_p, int64_t* out, void* stream) {
  if (!desc) return M3_ERR_NULL;
  if (desc->rows < 1 || desc->vocab < 1 || ld < desc->vocab) return M3_ERR_SHAPE;
  if (!dtype_ok(desc->dtype)) return M3_ERR_DTYPE;
  if (!logits || !uniform || !out) return M3_ERR_NULL;
  if (!aligned(logits, dsize(desc->dtype)) || !aligned(uniform, 4) || !aligned(temperature, 4) ||
      !aligned(top_k, 4) || !aligned(top_p, 4) || !aligned(min_p, 4) || !aligned(out, 8))
    return M3_ERR_ALIGN;
  if (desc->vocab > kMaxVocab) return M3_ERR_UNSUPPORTED;
  int rc = check_device();
  if (rc != M3_OK) return rc;
  SampleParams p;
  memset(&p, 0, sizeof(p));
  p.logits = logits; p.ld = ld; p.u = uniform;
  p.temperature = temperature; p.top_k = top_k; p.top_p = top_p; p.min_p = min_p;
  p.temperature0 = desc->temperature; p.top_k0 = desc->top_k; p.top_p0 = desc->top_p;
  p.min_p0 = desc->min_p;
  p.out = reinterpret_cast<long long*>(out);
  p.rows = desc->rows; p.V = desc->vocab; p.dtype = desc->dtype;
  p.shift = 50;   // the weights of a row add up to at most 2^62
  while (p.shift > 62 - 31 && (1LL << (62 - p.shift)) < desc->vocab) --p.shift;
  p.sms = device_sms();
  return status(launch_sample(p, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
