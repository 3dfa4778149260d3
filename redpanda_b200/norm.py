"""Layer norm and RMS norm on the sm_100a kernels, forward and backward.

* ``m3_layer_norm`` -- (x - mean) * rsqrt(var + eps) * weight + bias over the
  last dimension (the heads of redpanda/engine/search_mamba.py:60-83)
* ``m3_rms_norm`` -- x * rsqrt(mean(x^2) + eps) * weight (mamba.py:82-89)
* ``m3_add_rms_norm`` -- the residual's addition and the RMS norm behind it
  (mamba.py:591-595, 82-89): (norm(x + residual), x + residual)
* ``m3_rms_norm_8bit`` -- the RMS norm, with or without that addition, in 8 bits
  with a scale per row or group of columns, for a projection of 8-bit operands
* ``LayerNorm`` -- ``torch.nn.LayerNorm`` that runs ``m3_layer_norm`` on CUDA
  tensors when its class attribute ``use_kernel`` is set

float32 or bfloat16 activations, statistics and sums in float32, one rounding
of each output.  Each row is read once per pass; the weight gradients are summed
in a fixed order.  There is no CPU path: the functions raise on CPU tensors.
"""

import torch
import torch.nn as nn

from . import _lib
from . import _launch as H
from ._lib import AddNormDesc, Norm8Desc, NormDesc

MAX_D = 32768           # longest row of the kernels
_DENSE = torch.contiguous_format


def _forward(x2, ld, w, b, desc, out_dtype, stats):
    """y and, with ``stats``, one buffer of rstd and (layer norm) the means."""
    rows, d = x2.shape
    y = (torch.empty_like(x2) if out_dtype is x2.dtype and ld == d
         else torch.empty((rows, d), device=x2.device, dtype=out_dtype))
    st = (torch.empty((1 if desc.rms else 2, rows), device=x2.device, dtype=torch.float32)
          if stats else None)
    if rows:
        rstd = st.data_ptr() if stats else None
        mean = rstd + 4 * rows if stats and not desc.rms else None
        H.launch(x2.get_device(), _lib.load().m3_norm_fwd, desc, x2.data_ptr(), ld, w.data_ptr(),
                 H.ptr(b), y.data_ptr(), mean, rstd)
    return y, st


class _NormFn(torch.autograd.Function):
    """Rows of the norm with the analytic backward (m3_norm_fwd / m3_norm_bwd)."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps, rms, out_dtype):
        d = x.shape[-1]
        x2, ld = H.rows(x if x.dim() == 2 else x.reshape(-1, d))
        w = H.f32(weight)
        desc = NormDesc(x2.shape[0], d, H.code(x2.dtype), H.code(out_dtype), rms, eps)
        y, st = _forward(x2, ld, w, H.f32(bias), desc, out_dtype, True)
        H.save(ctx, x2, w, st)
        ctx.cfg = (ld, desc, out_dtype, x.shape, weight.dtype,
                   None if bias is None else bias.dtype)
        return y if x.dim() == 2 else y.view(x.shape)

    @staticmethod
    @H.once_differentiable
    def backward(ctx, g):
        x2, w, st = ctx.saved_tensors
        ld, desc, out_dtype, shape, wt, bt = ctx.cfg
        if ctx.hooked is not None or x2.stride(0) != ld:
            H.check_saved(ctx, (x2, w, st), g)
            (x2, ld), w, st = H.rows(x2), w.contiguous(), st.contiguous()
        if g.dtype is not out_dtype or not g.is_contiguous():
            g = g.to(out_dtype).contiguous()
        dx = torch.empty_like(x2, memory_format=torch.contiguous_format)
        dw = torch.empty_like(w)
        db = None if bt is None else torch.empty_like(w)
        rows = desc.rows
        if rows:
            lib = _lib.load()
            dev = x2.get_device()
            with H.on_device(dev):
                nws = lib.m3_norm_bwd_workspace_bytes(desc)
            ws = torch.empty(nws, device=x2.device, dtype=torch.uint8)
            rstd = st.data_ptr()
            H.launch(dev, lib.m3_norm_bwd, desc, x2.data_ptr(), ld, w.data_ptr(),
                     None if desc.rms else rstd + 4 * rows, rstd, g.data_ptr(), dx.data_ptr(),
                     dw.data_ptr(), H.ptr(db), ws.data_ptr(), nws)
        else:
            dw.zero_()
            if db is not None:
                db.zero_()
        return (dx if len(shape) == 2 else dx.view(shape), dw if wt is torch.float32 else dw.to(wt),
                db if bt is None or bt is torch.float32 else db.to(bt), None, None, None)


def _norm(name, x, weight, bias, eps, rms, out_dtype):
    d = x.shape[-1] if x.dim() else 0
    if d < 1 or weight.shape != (d,) or (bias is not None and bias.shape != (d,)):
        raise ValueError(f"{name}: weight (and bias) of the length of x's last dimension")
    if d > MAX_D:
        raise ValueError(f"{name}: rows of at most {MAX_D} elements")
    eps = float(eps)
    if not eps >= 0:
        raise ValueError(f"{name}: eps must not be negative")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    H.code(x.dtype), H.code(out_dtype)      # TypeError for another element type
    H.refuse_tangents(name, x, weight, bias)
    H.device_index(x, weight, bias)
    if H.needs_grad(x, weight, bias):
        return _NormFn.apply(x, weight, bias, eps, rms, out_dtype)
    x2, ld = H.rows(x if x.dim() == 2 else x.reshape(-1, d))
    desc = NormDesc(x2.shape[0], d, H.code(x2.dtype), H.code(out_dtype), rms, eps)
    y = _forward(x2, ld, H.f32(weight), H.f32(bias), desc, out_dtype, False)[0]
    return y if x.dim() == 2 else y.view(x.shape)


def m3_layer_norm(x, weight, bias=None, eps=1e-5, out_dtype=None):
    """Layer norm over the last dimension of x (..., d), d <= 32768.

    x float32 or bfloat16 (rows may be strided); weight and bias (d,) of any
    float type, used in float32; the result has ``out_dtype`` (default x's).
    Differentiable in x, weight and bias (once, in reverse mode)."""
    return _norm("m3_layer_norm", x, weight, bias, eps, 0, out_dtype)


def m3_rms_norm(x, weight, eps=1e-5, out_dtype=None):
    """x * rsqrt(mean(x^2) + eps) * weight over the last dimension; arguments as
    :func:`m3_layer_norm`."""
    return _norm("m3_rms_norm", x, weight, None, eps, 1, out_dtype)


def _add_forward(x2, lx, r2, lr, w, desc, out_dtype, stats):
    """(y, s, rstd or None) of rows."""
    s = torch.empty_like(r2, memory_format=_DENSE)
    y = torch.empty_like(r2, dtype=out_dtype, memory_format=_DENSE)
    rows = desc.rows
    st = torch.empty(rows, device=x2.device, dtype=torch.float32) if stats else None
    if rows:
        H.launch(x2.get_device(), _lib.load().m3_add_norm_fwd, desc, x2.data_ptr(), lx,
                 r2.data_ptr(), lr, w.data_ptr(), y.data_ptr(), s.data_ptr(),
                 st.data_ptr() if stats else None)
    return y, s, st


class _AddNormFn(torch.autograd.Function):
    """Addition and norm with the analytic backward (m3_add_norm_fwd / _bwd)."""

    @staticmethod
    def forward(ctx, x, residual, weight, eps, out_dtype):
        flat, d = x.dim() == 2, x.shape[-1]
        x2, lx = H.rows(x if flat else x.reshape(-1, d))
        r2, lr = H.rows(residual if flat else residual.reshape(-1, d))
        w = H.f32(weight)
        desc = AddNormDesc(x2.shape[0], d, H.code(x2.dtype), H.code(r2.dtype), H.code(out_dtype),
                           eps)
        y, s, st = _add_forward(x2, lx, r2, lr, w, desc, out_dtype, True)
        if not flat:
            y, s = y.view(x.shape), s.view(x.shape)
        H.save(ctx, s, w, st)
        ctx.cfg = (desc, x.dtype, out_dtype, weight.dtype)
        ctx.set_materialize_grads(False)
        return y, s

    @staticmethod
    @H.once_differentiable
    def backward(ctx, gy, gs):
        if gy is None and gs is None:
            return None, None, None, None, None
        desc, xt, yt, wt = ctx.cfg
        s, w, st = ts = ctx.saved_tensors
        ls = desc.d
        if ctx.hooked is not None:
            H.check_saved(ctx, ts, gs if gy is None else gy)
            s, w, st = s.contiguous(), w.contiguous(), st.contiguous()
        ty = s.dtype
        if gs is not None and (gs.dtype is not ty or not gs.is_contiguous()):
            gs = gs.to(ty).contiguous()
        if gy is None:      # the norm's result was not used
            return (gs if xt is ty else gs.to(xt)), gs, None, None, None
        if gy.dtype is not yt or not gy.is_contiguous():
            gy = gy.to(yt).contiguous()
        ds = torch.empty_like(s)
        dx = None if xt is ty else torch.empty_like(s, dtype=xt)
        dw = torch.empty_like(w)
        if desc.rows:
            lib = _lib.load()
            dev = s.get_device()
            with H.on_device(dev):
                nws = lib.m3_add_norm_bwd_workspace_bytes(desc)
            ws = w.new_empty(-(-nws // 4))
            H.launch(dev, lib.m3_add_norm_bwd, desc, s.data_ptr(), ls, w.data_ptr(),
                     st.data_ptr(), gy.data_ptr(), H.ptr(gs), ds.data_ptr(), H.ptr(dx),
                     dw.data_ptr(), ws.data_ptr(), nws)
        else:
            dw.zero_()
        return (ds if dx is None else dx), ds, (dw if wt is torch.float32 else dw.to(wt)), None, \
            None


def _check_rows(name, x, weight, residual, eps):
    shape = x.shape
    d = shape[-1] if shape else 0
    if d < 1 or weight.shape != shape[-1:]:
        raise ValueError(f"{name}: weight of the length of x's last dimension")
    if residual is not None and residual.shape != shape:
        raise ValueError(f"{name}: the residual has x's shape")
    if d > MAX_D:
        raise ValueError(f"{name}: rows of at most {MAX_D} elements")
    eps = float(eps)
    if not eps >= 0:
        raise ValueError(f"{name}: eps must not be negative")
    return d, eps


def m3_add_rms_norm(x, residual, weight, eps=1e-5, out_dtype=None):
    """(y, s): s = x + residual, the residual stream behind a layer, and y = its RMS
    norm, the next layer's input; x and residual (..., d), d <= 32768.

    x (a layer's output) and residual float32 or bfloat16 each, rows may be strided;
    s has the residual's element type, and y is the norm of s as rounded to it; y
    has ``out_dtype`` (default: the residual's).  weight (d,) of any float type,
    used in float32.  Differentiable in x, residual and weight (once, in reverse
    mode); the gradients of y and s reach x and the residual as one sum."""
    name = "m3_add_rms_norm"
    d, eps = _check_rows(name, x, weight, residual, eps)
    xt, st = x.dtype, residual.dtype
    out_dtype = st if out_dtype is None else out_dtype
    cx, cs, cy = H.code(xt), H.code(st), H.code(out_dtype)
    H.refuse_tangents(name, x, residual, weight)
    H.device_index(x, residual, weight)
    if H.needs_grad(x, residual, weight):
        return _AddNormFn.apply(x, residual, weight, eps, out_dtype)
    flat = x.dim() == 2
    x2, lx = H.rows(x if flat else x.reshape(-1, d))
    r2, lr = H.rows(residual if flat else residual.reshape(-1, d))
    y, s, _ = _add_forward(x2, lx, r2, lr, H.f32(weight),
                           AddNormDesc(x2.shape[0], d, cx, cs, cy, eps), out_dtype, False)
    return (y, s) if flat else (y.view(x.shape), s.view(x.shape))


def _grouped_rows(t, d, group):
    """H.rows of (..., d), copied where groups need vectors of 4 and it has none."""
    t2, ld = H.rows(t if t.dim() == 2 else t.reshape(-1, d))
    if group and (ld % 4 or t2.data_ptr() % (4 * t2.element_size())):
        t2, ld = t2.clone(memory_format=torch.contiguous_format), d
    return t2, ld


def m3_rms_norm_8bit(x, weight, residual=None, eps=1e-5, dtype=torch.float8_e4m3fn, group=None):
    """The RMS norm in 8 bits: (q, scale), or with ``residual`` (q, scale, s) where
    s = x + residual as in :func:`m3_add_rms_norm` and q is its norm.

    x (and residual) (..., d) float32 or bfloat16; ``dtype``: torch.float8_e4m3fn or
    torch.int8; ``group``: 32, 64 or 128 columns per scale (they have to divide d),
    or None, one scale per row.  q (..., d) and scale (..., 1) or (..., d / group)
    float32 stand for y = q * scale, with scale = max(max|y| / 448, 2^-126) (int8:
    127) over the group, y in float32, q = y / scale rounded to nearest even.  The
    scale is within 2^-23 of that and the quotient within 2^-22 before its rounding:
    next to the border of two codes either may come out.  A group with a NaN has the
    scale NaN.  Inference only."""
    name = "m3_rms_norm_8bit"
    d, eps = _check_rows(name, x, weight, residual, eps)
    cx = H.code(x.dtype)
    cs = cx if residual is None else H.code(residual.dtype)
    e4m3 = dtype is torch.float8_e4m3fn
    if not e4m3 and dtype is not torch.int8:
        raise TypeError(f"{name}: dtype is torch.float8_e4m3fn or torch.int8")
    if group is not None and (group not in (32, 64, 128) or d % group):
        raise ValueError(f"{name}: group is None, 32, 64 or 128 and divides d")
    if H.needs_grad(x, weight, residual):
        raise ValueError(f"{name} has no derivative: call it under torch.no_grad()")
    H.refuse_tangents(name, x, weight, residual)
    dev = H.device_index(x, weight, residual)
    x2, lx = _grouped_rows(x, d, group)
    q = torch.empty_like(x, dtype=dtype, memory_format=_DENSE)
    scale = x.new_empty((*x.shape[:-1], d // group if group else 1), dtype=torch.float32)
    s, r2, lr = None, None, 0
    if residual is not None:
        r2, lr = _grouped_rows(residual, d, group)
        s = torch.empty_like(residual, memory_format=_DENSE)
    rows = x2.shape[0]
    if rows:
        w = H.f32(weight)
        H.launch(dev, _lib.load().m3_norm8_fwd, Norm8Desc(rows, d, group or 0, cx, cs, e4m3, eps),
                 x2.data_ptr(), lx, H.ptr(r2), lr, w.data_ptr(), q.data_ptr(), scale.data_ptr(),
                 H.ptr(s))
    return (q, scale) if s is None else (q, scale, s)


class LayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` over one dimension; same parameters and state dict.

    ``use_kernel`` (class or instance attribute): run CUDA tensors of float32 or
    bfloat16 on :func:`m3_layer_norm`.  Off by default, where the forward is
    torch's own, bit for bit; the kernel's results differ by rounding (the order
    of its sums)."""

    use_kernel = False

    def forward(self, x):
        if (self.use_kernel and x.is_cuda and x.dtype in (torch.float32, torch.bfloat16)
                and self.weight is not None and len(self.normalized_shape) == 1
                and self.normalized_shape[0] <= MAX_D):
            # autocast: torch's layer norm gives float32 there
            wide = torch.float32 if torch.is_autocast_enabled("cuda") else None
            return m3_layer_norm(x, self.weight, self.bias, self.eps, out_dtype=wide)
        return super().forward(x)
