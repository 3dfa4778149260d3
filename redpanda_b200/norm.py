"""Layer norm and RMS norm on the sm_100a kernels, forward and backward.

* ``m3_layer_norm`` -- (x - mean) * rsqrt(var + eps) * weight + bias over the
  last dimension (the heads of redpanda/engine/search_mamba.py:60-83)
* ``m3_rms_norm`` -- x * rsqrt(mean(x^2) + eps) * weight (mamba.py:82-89)
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
from ._lib import NormDesc

MAX_D = 32768           # longest row of the kernels


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
