"""Host-side helpers of the operator modules: device, stream and row layout.

A call of a small operator costs more on the host than on the GPU, so these do
the least that is right: no device switch when the tensors are on the current
device, no copy or cast of what already has the kernels' layout and type.
"""

import contextlib

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import M3_BF16, M3_F32

_CODES = {torch.float32: M3_F32, torch.bfloat16: M3_BF16}
_HERE = contextlib.nullcontext()


def code(dtype):
    """The library's code of an element type."""
    c = _CODES.get(dtype)
    if c is None:
        raise TypeError(f"unsupported dtype {dtype}: float32 or bfloat16")
    return c


MAX_SIZE = 2 ** 30      # rows, steps and channels of one call (32-bit in the library)


def check_sizes(name, *sizes):
    if max(sizes) > MAX_SIZE:
        raise ValueError(f"{name}: sizes of at most {MAX_SIZE} each")


def device_index(*ts):
    """Index of the CUDA device that every tensor (None: skipped) is on."""
    dev = -1
    for t in ts:
        if t is None:
            continue
        i = t.get_device()
        if i < 0:
            raise RuntimeError("m3 ops run on CUDA tensors only (no CPU fallback)")
        if dev < 0:
            dev = i
        elif i != dev:
            raise RuntimeError("m3 ops need every tensor on one device")
    return dev


def on_device(index):
    """Context in which device ``index`` is the current one."""
    return _HERE if torch._C._cuda_getDevice() == index else torch.cuda.device(index)


def launch(index, fn, *args):
    """Call a library entry on device ``index`` and its current stream (the entry's
    last argument); raises for a status other than 0."""
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc)


def once_differentiable(body):
    """``torch.autograd.function.once_differentiable`` without its cost where no
    second derivative can follow (autograd is off while the backward runs)."""
    guarded = torch.autograd.function.once_differentiable(body)

    def backward(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else body(ctx, *grads)
    return backward


# the saved-tensor hooks in force, None without any
_hooks = getattr(torch._C._autograd, "_top_saved_tensors_default_hooks", lambda ignore: True)


def save(ctx, *ts):
    """Save tensors for the backward pass, and their types and shapes where hooks
    may give back others (``ctx.hooked``, else None)."""
    ctx.save_for_backward(*ts)
    ctx.hooked = None if _hooks(True) is None else [
        None if t is None else (t.dtype, t.shape) for t in ts]


def check_saved(ctx, ts, g):
    """Refuse saved tensors of another type, shape or device than forward; their
    layout may be another, and the caller looks at it again.  ``g``: the incoming
    gradient."""
    for t, like in zip(ts, ctx.hooked or ()):
        if t is not None and (t.dtype, t.shape) != like:
            raise RuntimeError("m3 ops: saved-tensor hooks have to give back the element type and "
                               "shape that they were given")
    device_index(g, *ts)


def f32(t):
    """A parameter as contiguous float32 (itself when it is)."""
    if t is None or (t.dtype is torch.float32 and t.is_contiguous()):
        return t
    return t.detach().to(torch.float32).contiguous()


def ptr(t):
    return None if t is None else t.data_ptr()


def refuse_tangents(name, *ts):
    """Raise for a tensor that carries a forward-mode tangent: the kernels have
    reverse-mode derivatives only, and would return a result without one."""
    if forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled():
        for t in ts:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError(f"{name} has no forward-mode derivative")


def needs_grad(*ts):
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


def seq_rows(t):
    """A (B, L, n) tensor whose rows (b, t) have one stride, and that stride."""
    B, L, n = t.shape
    if t.is_contiguous():
        return t, n
    s0, s1, s2 = t.stride()
    if s2 == 1 and (L == 1 or B == 1 or s0 == L * s1):
        ld = s1 if L > 1 else s0 if B > 1 else n
        if ld >= n:
            return t, ld
    return t.contiguous(), n


def rows(t):
    """The same for (rows, n)."""
    r, n = t.shape
    if t.is_contiguous():
        return t, n
    s0, s1 = t.stride()
    if s1 == 1 and (r == 1 or s0 >= n):
        return t, (s0 if r > 1 else n)
    return t.contiguous(), n
