"""The short causal convolution and the selective scan on the sm_100a kernels.

The pair that a selective state space layer is made of, beside the trapezoidal
scan of :mod:`redpanda_b200.scan`:

* ``m3_causal_conv`` / ``m3_causal_conv_with_state`` -- one filter of up to 8
  taps per channel over time, with silu; prompts and training
* ``m3_causal_conv_step_`` -- one token, the state moved up in place
* ``m3_selective_scan`` / ``m3_selective_scan_with_state`` --
  h_t = exp(de_t A) h_{t-1} + de_t u_t B_t, y_t = (C_t . h_t + D u_t) silu(z_t),
  de = softplus(dt + dt_bias); prompts and training
* ``m3_selective_step_`` -- one token, in place on h

Tensors are (B, L, channels), float32 or bfloat16, and may be row-strided views
(a half of in_proj's output, columns of x_proj's); states are the convolution's
last K-1 input rows (B, K-1, D) in x's element type and h (B, D, N) float32.
``lengths`` (B,) gives a padded batch's true lengths, from 0 to L: steps at or
past a row's length are not read, their outputs and gradients are zero, and the
state is the one at the length.  Arithmetic and states are float32, each output
is rounded once, and sums run in a fixed order.  Outputs are differentiable
(once, in reverse mode); the states are not, neither as input nor as output.
There is no CPU path: every op raises on CPU tensors.
"""

import torch
from torch.autograd.graph import increment_version

from . import _lib
from . import _launch as H
from ._lib import ConvDesc, SelArgs, SelDesc, SelGrads

MAX_WIDTH = 8           # taps of the convolution
MAX_STATE = 128         # states per channel of the selective scan


def _common(*ts):
    """One element type for the activations: theirs when they agree, else float32."""
    dt = None
    for t in ts:
        if t is None or t.dtype is dt:
            continue
        H.code(t.dtype)      # TypeError for another element type
        dt = t.dtype if dt is None else torch.float32
    return dt


def _lengths(name, lengths, B):
    if lengths is None:
        return None
    if lengths.shape != (B,) or lengths.dtype.is_floating_point or lengths.dtype is torch.bool:
        raise ValueError(f"{name}: lengths are (B,) integers")
    if lengths.dtype is not torch.int32:
        lengths = lengths.to(torch.int64).clamp(0, 2 ** 31 - 1).to(torch.int32)
    return lengths.contiguous()


def _fixed_state(name, state):
    if H.needs_grad(state):
        raise ValueError(f"{name}: the state is not differentiable (detach it)")


def _typed(t, dtype):
    return t if t is None or t.dtype is dtype else t.to(dtype)


def _contiguous(ts):
    return [None if t is None else t.contiguous() for t in ts]


# ---------------------------------------------------------------- convolution

def _check_filter(name, D, weight, bias):
    if weight.dim() != 2 or weight.shape[0] != D or not 1 <= weight.shape[1] <= MAX_WIDTH:
        raise ValueError(f"{name}: weight is (D, K) with K from 1 to {MAX_WIDTH}")
    if bias is not None and bias.shape != (D,):
        raise ValueError(f"{name}: bias is (D,)")


def _check_conv(name, x, weight, bias, state, lengths):
    if x.dim() != 3 or x.shape[-1] < 1:
        raise ValueError(f"{name}: x is (B, L, D)")
    H.code(x.dtype)
    B, L, D = x.shape
    H.check_sizes(name, B, L, D)
    _check_filter(name, D, weight, bias)
    if state is not None and (state.shape != (B, weight.shape[1] - 1, D)
                              or state.dtype is not x.dtype):
        raise ValueError(f"{name}: the state is (B, K - 1, D) in x's element type")
    _fixed_state(name, state)
    lens = _lengths(name, lengths, B)
    H.refuse_tangents(name, x, weight, bias, state)
    H.device_index(x, weight, bias, state, lens)
    return lens


def _conv_fwd(x, ld, w, b, state, lengths, silu, want_state):
    B, L, D = x.shape
    K = w.shape[1]
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    out = torch.empty((B, K - 1, D), device=x.device, dtype=x.dtype) if want_state else None
    if B == 0 or L == 0:
        if out is not None:
            out.copy_(state) if state is not None else out.zero_()
        return y, out
    H.launch(x.get_device(), _lib.load().m3_causal_conv_fwd,
             ConvDesc(B, L, D, K, H.code(x.dtype), silu), x.data_ptr(), ld, w.data_ptr(), H.ptr(b),
             H.ptr(state), H.ptr(lengths), y.data_ptr(), H.ptr(out))
    return y, out


class _ConvFn(torch.autograd.Function):
    """The causal convolution with its backward (m3_causal_conv_fwd / _bwd)."""

    @staticmethod
    def forward(ctx, x, weight, bias, state, lengths, silu, want_state):
        x2, ld = H.seq_rows(x)
        w, b = H.f32(weight), H.f32(bias)
        st = None if state is None else state.contiguous()
        y, out = _conv_fwd(x2, ld, w, b, st, lengths, silu, want_state)
        H.save(ctx, x2, w, b, st, lengths)
        ctx.cfg = (ld, silu, weight.dtype, None if bias is None else bias.dtype)
        ctx.set_materialize_grads(False)
        if out is not None:
            ctx.mark_non_differentiable(out)
        return y, out

    @staticmethod
    @H.once_differentiable
    def backward(ctx, g, _):
        if g is None:
            return (None,) * 7
        x, w, b, state, lengths = ts = ctx.saved_tensors
        ld, silu, wt, bt = ctx.cfg
        if ctx.hooked is not None or x.stride(1) != ld:
            H.check_saved(ctx, ts, g)
            x, ld = H.seq_rows(x)
            w, b, state, lengths = _contiguous(ts[1:])
        B, L, D = x.shape
        K = w.shape[1]
        if g.dtype is not x.dtype or not g.is_contiguous():
            g = g.to(x.dtype).contiguous()
        dx = torch.empty_like(x, memory_format=torch.contiguous_format)
        dw = torch.empty_like(w)
        db = None if b is None else torch.empty_like(b)
        if B == 0 or L == 0:
            dw.zero_()
            if db is not None:
                db.zero_()
        else:
            lib = _lib.load()
            dev = x.get_device()
            desc = ConvDesc(B, L, D, K, H.code(x.dtype), silu)
            with H.on_device(dev):
                nws = lib.m3_causal_conv_bwd_workspace_bytes(desc)
            ws = torch.empty(nws, device=x.device, dtype=torch.uint8)
            H.launch(dev, lib.m3_causal_conv_bwd, desc, x.data_ptr(), ld, w.data_ptr(), H.ptr(b),
                     H.ptr(state), H.ptr(lengths), g.data_ptr(), dx.data_ptr(), dw.data_ptr(),
                     H.ptr(db), ws.data_ptr(), nws)
        return dx, _typed(dw, wt), _typed(db, bt), None, None, None, None


def _conv(name, x, weight, bias, silu, state, lengths, want_state):
    lens = _check_conv(name, x, weight, bias, state, lengths)
    if H.needs_grad(x, weight, bias):
        return _ConvFn.apply(x, weight, bias, state, lens, int(silu), want_state)
    x2, ld = H.seq_rows(x)
    st = None if state is None else state.contiguous()
    return _conv_fwd(x2, ld, H.f32(weight), H.f32(bias), st, lens, int(silu), want_state)


def m3_causal_conv(x, weight, bias=None, silu=True, state=None, lengths=None):
    """y[b, t] = act(bias + sum_k weight[:, k] * x[b, t - K + 1 + k]), (B, L, D).

    weight (D, K), K <= 8; ``silu``: act is silu, else nothing; ``state``
    (B, K - 1, D): the input rows before x, oldest first (zeros when None);
    ``lengths`` (B,): see the module.  Differentiable in x, weight and bias."""
    return _conv("m3_causal_conv", x, weight, bias, silu, state, lengths, False)[0]


def m3_causal_conv_with_state(x, weight, bias=None, silu=True, state=None, lengths=None):
    """:func:`m3_causal_conv` and the new state: (y, (B, K - 1, D)), the last
    K - 1 rows of [state; x[:length]], for :func:`m3_causal_conv_step_` or the
    next part of the sequence."""
    return _conv("m3_causal_conv_with_state", x, weight, bias, silu, state, lengths, True)


def m3_causal_conv_step_(state, x_t, weight, bias=None, silu=True):
    """One token per row: y (B, D) from [state; x_t]; ``state`` (B, K - 1, D),
    contiguous and in x_t's element type, moves up by one row IN PLACE.
    Inference only."""
    name = "m3_causal_conv_step_"
    if H.needs_grad(state, x_t, weight, bias):
        raise ValueError(f"{name} works in place: call it under torch.no_grad()")
    if x_t.dim() != 2 or x_t.shape[1] < 1:
        raise ValueError(f"{name}: x_t is (B, D)")
    B, D = x_t.shape
    H.check_sizes(name, B, D)
    _check_filter(name, D, weight, bias)
    K = weight.shape[1]
    if state.shape != (B, K - 1, D) or state.dtype is not x_t.dtype or not state.is_contiguous():
        raise ValueError(f"{name}: the state is (B, K - 1, D), contiguous (it is updated in "
                         "place) and of x_t's element type")
    code = H.code(x_t.dtype)
    H.refuse_tangents(name, x_t, state, weight, bias)
    dev = H.device_index(x_t, state, weight, bias)
    y = torch.empty_like(x_t, memory_format=torch.contiguous_format)
    if B == 0:
        return y
    x2, ld = H.rows(x_t)
    w, b = H.f32(weight), H.f32(bias)
    H.launch(dev, _lib.load().m3_causal_conv_step, ConvDesc(B, 1, D, K, code, int(silu)),
             state.data_ptr(), x2.data_ptr(), ld, w.data_ptr(), H.ptr(b), y.data_ptr())
    increment_version(state)    # a backward pass that has saved it raises
    return y


# ---------------------------------------------------------------- scan

def _check_params(name, D, A, Dskip, dt_bias):
    if A.dim() != 2 or A.shape[0] != D or not 1 <= A.shape[1] <= MAX_STATE:
        raise ValueError(f"{name}: A is (D, N) with N from 1 to {MAX_STATE}")
    for t, what in ((Dskip, "D"), (dt_bias, "dt_bias")):
        if t is not None and t.shape != (D,):
            raise ValueError(f"{name}: {what} is (D,)")


def _sel_args(prepared, A, Dskip, dt_bias, state, lengths):
    """SelArgs of the prepared (tensor, row stride) pairs u, dt, z, B, C."""
    (u, lu), (dt, ld), (z, lz), (Bm, lb), (Cm, lc) = prepared
    return SelArgs(u.data_ptr(), lu, dt.data_ptr(), ld, H.ptr(z), lz, Bm.data_ptr(), lb,
                   Cm.data_ptr(), lc, A.data_ptr(), H.ptr(Dskip), H.ptr(dt_bias), H.ptr(state),
                   H.ptr(lengths))


def _scan_fwd(prepared, A, Dskip, dt_bias, state, lengths, softplus, want_state, want_ckpt):
    u = prepared[0][0]
    dev = u.get_device()
    B, L, D = u.shape
    N = A.shape[1]
    y = torch.empty_like(u, memory_format=torch.contiguous_format)
    h = torch.empty((B, D, N), device=u.device, dtype=torch.float32) if want_state else None
    if B == 0 or L == 0:
        if h is not None:
            h.copy_(state) if state is not None else h.zero_()
        return y, h, None
    lib = _lib.load()
    desc = SelDesc(B, L, D, N, H.code(u.dtype), softplus)
    ckpt = ws = None
    with H.on_device(dev):
        if want_ckpt:
            nck = lib.m3_selective_ckpt_floats(desc)
            ckpt = torch.empty(nck, device=u.device, dtype=torch.float32) if nck else None
        nws = lib.m3_selective_fwd_workspace_bytes(desc)
    if nws:
        ws = torch.empty(nws, device=u.device, dtype=torch.uint8)
    H.launch(dev, lib.m3_selective_fwd, desc,
             _sel_args(prepared, A, Dskip, dt_bias, state, lengths), y.data_ptr(), H.ptr(h),
             H.ptr(ckpt), H.ptr(ws), nws)
    return y, h, ckpt


def _prepare(seq, u, dt, z, Bm, Cm):
    """(tensor, row stride) of each activation in their common element type."""
    ty = _common(u, dt, z, Bm, Cm)
    return [(None, 0) if t is None else seq(_typed(t, ty)) for t in (u, dt, z, Bm, Cm)]


class _SelectiveScanFn(torch.autograd.Function):
    """The selective scan with its analytic backward (m3_selective_fwd / _bwd)."""

    @staticmethod
    def forward(ctx, u, dt, A, Bm, Cm, Dskip, z, dt_bias, state, lengths, softplus, want_state):
        prepared = _prepare(H.seq_rows, u, dt, z, Bm, Cm)
        a32, d32, b32, st = H.f32(A), H.f32(Dskip), H.f32(dt_bias), H.f32(state)
        y, h, ckpt = _scan_fwd(prepared, a32, d32, b32, st, lengths, softplus, want_state, True)
        H.save(ctx, *(t for t, _ in prepared), a32, d32, b32, st, lengths, ckpt)
        ctx.cfg = ([ld for _, ld in prepared], softplus,
                   [None if t is None else t.dtype for t in (u, dt, A, Bm, Cm, Dskip, z, dt_bias)])
        ctx.set_materialize_grads(False)
        if h is not None:
            ctx.mark_non_differentiable(h)
        return y, h

    @staticmethod
    @H.once_differentiable
    def backward(ctx, g, _):
        if g is None:
            return (None,) * 12
        ts = ctx.saved_tensors
        lds, softplus, types = ctx.cfg
        if ctx.hooked is not None or any(t is not None and t.stride(1) != ld
                                         for t, ld in zip(ts, lds)):
            H.check_saved(ctx, ts, g)
            seqs, lds = zip(*((None, 0) if t is None else H.seq_rows(t) for t in ts[:5]))
            ts = (*seqs, *_contiguous(ts[5:]))
        u, dt, z, Bm, Cm, A, Dskip, dt_bias, state, lengths, ckpt = ts
        B, L, D = u.shape
        N = A.shape[1]
        dev, ty = u.device, u.dtype
        if g.dtype is not ty or not g.is_contiguous():
            g = g.to(ty).contiguous()
        fresh = torch.contiguous_format
        du = torch.empty_like(u, memory_format=fresh)
        ddt = torch.empty_like(u, memory_format=fresh)
        dz = None if z is None else torch.empty_like(u, memory_format=fresh)
        dB = torch.empty_like(Bm, memory_format=fresh)
        dC = torch.empty_like(Cm, memory_format=fresh)
        dA = torch.empty_like(A)
        dD = None if Dskip is None else torch.empty_like(Dskip)
        dbias = None if dt_bias is None else torch.empty_like(dt_bias)
        if B == 0 or L == 0:
            for t in (dA, dD, dbias):
                if t is not None:
                    t.zero_()
        else:
            lib = _lib.load()
            desc = SelDesc(B, L, D, N, H.code(ty), softplus)
            args = _sel_args(tuple(zip((u, dt, z, Bm, Cm), lds)), A, Dskip, dt_bias, state, lengths)
            grads = SelGrads(du.data_ptr(), ddt.data_ptr(), H.ptr(dz), dB.data_ptr(),
                             dC.data_ptr(), dA.data_ptr(), H.ptr(dD), H.ptr(dbias))
            index = u.get_device()
            with H.on_device(index):
                nws = lib.m3_selective_bwd_workspace_bytes(desc)
            ws = torch.empty(nws, device=dev, dtype=torch.uint8)
            H.launch(index, lib.m3_selective_bwd, desc, args, g.data_ptr(), H.ptr(ckpt), grads,
                     ws.data_ptr(), nws)
        out = (du, ddt, dA, dB, dC, dD, dz, dbias)
        return (*(_typed(t, ty) for t, ty in zip(out, types)), None, None, None, None)


def _scan(name, u, dt, A, Bm, Cm, D, z, dt_bias, softplus, state, lengths, want_state):
    if u.dim() != 3 or u.shape[-1] < 1 or dt.shape != u.shape or \
            (z is not None and z.shape != u.shape):
        raise ValueError(f"{name}: u, dt and z are (B, L, D)")
    B, L, d = u.shape
    H.check_sizes(name, B, L, d)
    _check_params(name, d, A, D, dt_bias)
    N = A.shape[1]
    if Bm.shape != (B, L, N) or Cm.shape != (B, L, N):
        raise ValueError(f"{name}: B and C are (B, L, N) with A's N")
    if state is not None and state.shape != (B, d, N):
        raise ValueError(f"{name}: the state is (B, D, N)")
    _common(u, dt, z, Bm, Cm)
    _fixed_state(name, state)
    lens = _lengths(name, lengths, B)
    H.refuse_tangents(name, u, dt, A, Bm, Cm, D, z, dt_bias, state)
    H.device_index(u, dt, A, Bm, Cm, D, z, dt_bias, state, lens)
    if H.needs_grad(u, dt, A, Bm, Cm, D, z, dt_bias):
        return _SelectiveScanFn.apply(u, dt, A, Bm, Cm, D, z, dt_bias, state, lens, int(softplus),
                                      want_state)
    return _scan_fwd(_prepare(H.seq_rows, u, dt, z, Bm, Cm), H.f32(A), H.f32(D), H.f32(dt_bias),
                     H.f32(state), lens, int(softplus), want_state, False)[:2]


def m3_selective_scan(u, dt, A, Bm, Cm, D=None, z=None, dt_bias=None, softplus=True, state=None,
                      lengths=None):
    """y (B, L, D) of the selective scan over u, dt (B, L, D), A (D, N), Bm, Cm
    (B, L, N); N <= 128.

    ``D`` (D,): the skip weight; ``z`` (B, L, D): the gate; ``dt_bias`` (D,) is
    added to dt before softplus (``softplus=False``: the sum is the step size);
    ``state`` (B, D, N): the state before the first step (zero when None);
    ``lengths`` (B,): see the module.  u, dt, z, Bm and Cm of one element type
    (float32 when they differ), which is y's.  Differentiable in all but the
    state."""
    return _scan("m3_selective_scan", u, dt, A, Bm, Cm, D, z, dt_bias, softplus, state, lengths,
                 False)[0]


def m3_selective_scan_with_state(u, dt, A, Bm, Cm, D=None, z=None, dt_bias=None, softplus=True,
                                 state=None, lengths=None):
    """:func:`m3_selective_scan` and the state h (B, D, N) float32 at each row's
    length, for :func:`m3_selective_step_` or the next part of the sequence."""
    return _scan("m3_selective_scan_with_state", u, dt, A, Bm, Cm, D, z, dt_bias, softplus, state,
                 lengths, True)


def m3_selective_step_(h, u_t, dt_t, A, B_t, C_t, D=None, z=None, dt_bias=None, softplus=True):
    """One token per row, updating ``h`` (B, D, N) float32 contiguous IN PLACE;
    u_t, dt_t, z (B, D), B_t, C_t (B, N); returns y (B, D).  At most 524280 rows.
    Inference only."""
    name = "m3_selective_step_"
    if H.needs_grad(h, u_t, dt_t, A, B_t, C_t, D, z, dt_bias):
        raise ValueError(f"{name} works in place: call it under torch.no_grad()")
    if u_t.dim() != 2 or u_t.shape[1] < 1 or dt_t.shape != u_t.shape or \
            (z is not None and z.shape != u_t.shape):
        raise ValueError(f"{name}: u_t, dt_t and z are (B, D)")
    B, d = u_t.shape
    H.check_sizes(name, B, d)
    _check_params(name, d, A, D, dt_bias)
    N = A.shape[1]
    if B_t.shape != (B, N) or C_t.shape != (B, N):
        raise ValueError(f"{name}: B_t and C_t are (B, N) with A's N")
    if h.shape != (B, d, N) or h.dtype is not torch.float32 or not h.is_contiguous():
        raise ValueError(f"{name}: h is (B, D, N), float32 and contiguous (it is updated in place)")
    ty = _common(u_t, dt_t, z, B_t, C_t)
    H.refuse_tangents(name, h, u_t, dt_t, A, B_t, C_t, D, z, dt_bias)
    dev = H.device_index(h, u_t, dt_t, A, B_t, C_t, D, z, dt_bias)
    u2, lu = H.rows(_typed(u_t, ty))
    d2, ld = H.rows(_typed(dt_t, ty))
    z2, lz = (None, 0) if z is None else H.rows(_typed(z, ty))
    b2, lb = H.rows(_typed(B_t, ty))
    c2, lc = H.rows(_typed(C_t, ty))
    y = torch.empty_like(u2, memory_format=torch.contiguous_format)
    if B == 0:
        return y
    a32, d32, b32 = H.f32(A), H.f32(D), H.f32(dt_bias)
    args = SelArgs(u2.data_ptr(), lu, d2.data_ptr(), ld, H.ptr(z2), lz, b2.data_ptr(), lb,
                   c2.data_ptr(), lc, a32.data_ptr(), H.ptr(d32), H.ptr(b32), None, None)
    H.launch(dev, _lib.load().m3_selective_step, SelDesc(B, 1, d, N, H.code(ty), int(softplus)),
             args, h.data_ptr(), y.data_ptr())
    increment_version(h)
    return y
