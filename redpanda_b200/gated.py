"""The gated linear recurrence on the sm_100a kernels.

A diagonal recurrence with a decay that each token sets, beside the scans of
:mod:`redpanda_b200.scan` and :mod:`redpanda_b200.selective` (which keep N states
per channel; this one keeps one):

* ``m3_gated_scan`` / ``m3_gated_scan_with_state`` --
  a_t = exp(-c softplus(decay) sigmoid(rgate_t)),
  h_t = a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(igate_t) x_t, y = h;
  prompts and training
* ``m3_gated_step_`` -- one token, in place on h

Tensors are (B, L, D), float32 or bfloat16, and may be row-strided views (halves
of a projection's output); the state is h (B, D) float32.  ``lengths`` (B,) gives
a padded batch's true lengths, from 0 to L: steps at or past a row's length are
not read, their outputs and gradients are zero, and the state is the one at the
length.  Arithmetic and states are float32, each output is rounded once, and sums
run in a fixed order.  Outputs are differentiable (once, in reverse mode); the
states are not, neither as input nor as output.  There is no CPU path: every op
raises on CPU tensors.
"""

import math

import torch
from torch.autograd.graph import increment_version

from . import _lib
from . import _launch as H
from ._lib import GatedArgs, GatedDesc
from .selective import _common, _contiguous, _fixed_state, _lengths, _typed


def _args(prepared, decay, state, lengths):
    (x, lx), (r, lr), (i, li) = prepared
    return GatedArgs(x.data_ptr(), lx, r.data_ptr(), lr, i.data_ptr(), li, decay.data_ptr(),
                     H.ptr(state), H.ptr(lengths))


def _forward(prepared, decay, c, state, lengths, want_state, want_ckpt):
    x = prepared[0][0]
    B, L, D = x.shape
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    h = decay.new_empty(B, D) if want_state else None
    if B == 0 or L == 0:
        if h is not None:
            h.copy_(state) if state is not None else h.zero_()
        return y, h, None
    lib = _lib.load()
    desc = GatedDesc(B, L, D, H.code(x.dtype), c)
    ckpt = decay.new_empty(lib.m3_gated_ckpt_floats(desc)) if want_ckpt else None
    H.launch(x.get_device(), lib.m3_gated_fwd, desc, _args(prepared, decay, state, lengths),
             y.data_ptr(), H.ptr(h), H.ptr(ckpt))
    return y, h, ckpt


def _prepare(seq, x, r, i):
    """(tensor, row stride) of each activation in their common element type."""
    ty = x.dtype
    if r.dtype is not ty or i.dtype is not ty:
        ty = torch.float32
        x, r, i = _typed(x, ty), _typed(r, ty), _typed(i, ty)
    return seq(x), seq(r), seq(i)


class _GatedScanFn(torch.autograd.Function):
    """The recurrence with its analytic backward (m3_gated_fwd / _bwd)."""

    @staticmethod
    def forward(ctx, x, rgate, igate, decay, c, state, lengths, want_state):
        prepared = _prepare(H.seq_rows, x, rgate, igate)
        d32, st = H.f32(decay), H.f32(state)
        y, h, ckpt = _forward(prepared, d32, c, st, lengths, want_state, True)
        H.save(ctx, *(t for t, _ in prepared), d32, lengths, ckpt)
        ctx.cfg = ([ld for _, ld in prepared], c, [t.dtype for t in (x, rgate, igate, decay)])
        ctx.set_materialize_grads(False)
        if h is not None:
            ctx.mark_non_differentiable(h)
        return y, h

    @staticmethod
    @H.once_differentiable
    def backward(ctx, g, _):
        if g is None:
            return (None,) * 8
        ts = ctx.saved_tensors
        lds, c, types = ctx.cfg
        if ctx.hooked is not None or any(t.stride(1) != ld for t, ld in zip(ts, lds)):
            H.check_saved(ctx, ts, g)
            seqs, lds = zip(*(H.seq_rows(t) for t in ts[:3]))
            ts = (*seqs, *_contiguous(ts[3:]))
        x, r, i, decay, lengths, ckpt = ts
        B, L, D = x.shape
        ty = x.dtype
        if g.dtype is not ty or not g.is_contiguous():
            g = g.to(ty).contiguous()
        grads = [torch.empty_like(x, memory_format=torch.contiguous_format) for _ in range(3)]
        ddecay = torch.empty_like(decay)
        if B == 0 or L == 0:
            ddecay.zero_()
        else:
            lib = _lib.load()
            index = x.get_device()
            desc = GatedDesc(B, L, D, H.code(ty), c)
            with H.on_device(index):
                nws = lib.m3_gated_bwd_workspace_bytes(desc)
            ws = decay.new_empty(-(-nws // 4))
            # the checkpoints hold what the state before x was
            H.launch(index, lib.m3_gated_bwd, desc,
                     _args(tuple(zip((x, r, i), lds)), decay, None, lengths), g.data_ptr(),
                     ckpt.data_ptr(), *(t.data_ptr() for t in grads), ddecay.data_ptr(),
                     ws.data_ptr(), nws)
        return (*(_typed(t, ty) for t, ty in zip((*grads, ddecay), types)), None, None, None, None)


def _check(name, x, rgate, igate, decay, c, dims):
    shape = x.shape
    if len(shape) != dims or shape[-1] < 1 or rgate.shape != shape or igate.shape != shape:
        what = "(B, L, D)" if dims == 3 else "(B, D)"
        raise ValueError(f"{name}: x, rgate and igate are {what}")
    H.check_sizes(name, *shape)
    if decay.shape != shape[-1:]:
        raise ValueError(f"{name}: decay is (D,)")
    c = float(c)
    if not 0 < c < math.inf:
        raise ValueError(f"{name}: c must be positive and finite")
    _common(x, rgate, igate)
    return c


def _scan(name, x, rgate, igate, decay, c, state, lengths, want_state):
    c = _check(name, x, rgate, igate, decay, c, 3)
    B, _, D = x.shape
    if state is not None and state.shape != (B, D):
        raise ValueError(f"{name}: the state is (B, D)")
    _fixed_state(name, state)
    lens = _lengths(name, lengths, B)
    H.refuse_tangents(name, x, rgate, igate, decay, state)
    H.device_index(x, rgate, igate, decay, state, lens)
    if H.needs_grad(x, rgate, igate, decay):
        return _GatedScanFn.apply(x, rgate, igate, decay, c, state, lens, want_state)
    return _forward(_prepare(H.seq_rows, x, rgate, igate), H.f32(decay), c, H.f32(state), lens,
                    want_state, False)[:2]


def m3_gated_scan(x, rgate, igate, decay, c=8.0, state=None, lengths=None):
    """y (B, L, D) of the gated linear recurrence over x, rgate, igate (B, L, D)
    and decay (D,).

    ``rgate`` and ``igate``: the recurrence's and the input's gate before their
    sigmoids; ``decay``: a = exp(-c softplus(decay)) with the gate fully open;
    ``state`` (B, D): the state before the first step (zero when None);
    ``lengths`` (B,): see the module.  x and the gates of one element type (float32
    when they differ), which is y's.  Differentiable in x, the gates and decay."""
    return _scan("m3_gated_scan", x, rgate, igate, decay, c, state, lengths, False)[0]


def m3_gated_scan_with_state(x, rgate, igate, decay, c=8.0, state=None, lengths=None):
    """:func:`m3_gated_scan` and the state h (B, D) float32 at each row's length,
    for :func:`m3_gated_step_` or the next part of the sequence."""
    return _scan("m3_gated_scan_with_state", x, rgate, igate, decay, c, state, lengths, True)


def m3_gated_step_(h, x_t, rgate_t, igate_t, decay, c=8.0):
    """One token per row, updating ``h`` (B, D) float32 contiguous IN PLACE; x_t
    and the gates (B, D); returns y (B, D), h in their element type.  Inference
    only."""
    name = "m3_gated_step_"
    if H.needs_grad(h, x_t, rgate_t, igate_t, decay):
        raise ValueError(f"{name} works in place: call it under torch.no_grad()")
    c = _check(name, x_t, rgate_t, igate_t, decay, c, 2)
    shape = x_t.shape
    if h.shape != shape or h.dtype is not torch.float32 or not h.is_contiguous():
        raise ValueError(f"{name}: h is (B, D), float32 and contiguous (it is updated in place)")
    H.refuse_tangents(name, h, x_t, rgate_t, igate_t, decay)
    dev = H.device_index(h, x_t, rgate_t, igate_t, decay)
    prepared = _prepare(H.rows, x_t, rgate_t, igate_t)
    x = prepared[0][0]
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    B, D = shape
    if B == 0:
        return y
    d32 = H.f32(decay)
    H.launch(dev, _lib.load().m3_gated_step, GatedDesc(B, 1, D, H.code(x.dtype), c),
             _args(prepared, d32, None, None), h.data_ptr(), y.data_ptr())
    increment_version(h)
    return y
