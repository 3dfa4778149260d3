"""Projections of few rows with 4-bit weights on the sm_100a kernels.

* ``Q4Weight`` -- a weight (d_out, d_in) as 4-bit codes with a scale, and a center,
  per group of 32, 64 or 128 columns, laid out once for the kernel
* ``m3_rows_linear_q4`` -- :func:`redpanda_b200.scan.m3_rows_linear` with such a
  weight: at most 8 rows, the RMS norm, bias, silu and residual folded in

The rows are float32 or bfloat16; products and sums are float32 on unrounded
inputs, and each output is rounded once.  There is no CPU path: the product raises
on CPU tensors (a ``Q4Weight`` may be made on the CPU and moved).
"""

import torch
from torch.autograd.graph import increment_version

from . import _lib
from . import _launch as H
from ._lib import RowsQ4Desc

MAX_ROWS = 8            # rows of one product
MAX_IN = 65536          # columns of a weight
GROUPS = (32, 64, 128)


class Q4Weight:
    """w[o, k] = scale[o, k // group] * (code[o, k] - 8) + center[o, k // group].

    Codes are whole numbers from 0 to 15; scale and center are held in bfloat16
    (given in another type they are rounded to it); without centers they are 0.
    Make one with :meth:`quantize`, :meth:`from_codes` or :meth:`from_packed`.
    ``d_out``, ``d_in``, ``group``, ``device`` and ``has_center`` say what it is;
    :meth:`dequantize` gives the weight it stands for."""

    def __init__(self, codes, scales, d_out, d_in, group, has_center):
        self.codes, self.scales = codes, scales      # laid out as m3_rows_linear_q4 reads them
        self.d_out, self.d_in, self.group, self.has_center = d_out, d_in, group, has_center

    @property
    def device(self):
        return self.codes.device

    def to(self, device):
        return Q4Weight(self.codes.to(device), self.scales.to(device), self.d_out, self.d_in,
                        self.group, self.has_center)

    @staticmethod
    def _check(shape, group):
        if group not in GROUPS:
            raise ValueError(f"Q4Weight: group is one of {GROUPS}")
        if len(shape) != 2 or min(shape) < 1:
            raise ValueError("Q4Weight: a weight is (d_out, d_in)")
        if shape[1] > MAX_IN:
            raise ValueError(f"Q4Weight: at most {MAX_IN} columns")
        H.check_sizes("Q4Weight", *shape)

    @classmethod
    def quantize(cls, weight, group=64, center=True):
        """Nearest codes of ``weight`` (d_out, d_in): with ``center`` a group's
        smallest and largest weight get the codes 0 and 15, without, the largest
        magnitude gets 1 or 15.  The weights have to be finite."""
        cls._check(weight.shape, group)
        w = weight.detach().to(torch.float32)
        if not bool(torch.isfinite(w).all()):
            raise ValueError("Q4Weight: weights have to be finite")
        d_out, d_in = w.shape
        n = -(-d_in // group)
        # the last group's missing columns as copies of its last: they change no extreme
        w = torch.cat([w, w[:, -1:].expand(d_out, n * group - d_in)], 1).view(d_out, n, group)
        lo, hi = w.amin(2), w.amax(2)
        tiny = torch.finfo(torch.float32).tiny
        if center:
            scale = (hi / 15 - lo / 15).to(torch.bfloat16)
            mid = (lo + 8 * scale.float()).to(torch.bfloat16)
            off = mid.float()
        else:
            scale = torch.maximum(hi / 7, -lo / 8).to(torch.bfloat16)
            mid, off = None, torch.zeros_like(lo)
        q = (w - off[..., None]) / scale.float().clamp(min=tiny)[..., None]
        q = q.round_().add_(8).clamp_(0, 15).to(torch.uint8).view(d_out, n * group)[:, :d_in]
        return cls.from_codes(q, scale, mid, group)

    @classmethod
    def from_packed(cls, packed, scale, center=None, d_in=None, group=64):
        """From codes two to a byte, (d_out, ceil(d_in / 2)) uint8, the even column
        in the low half; the rest as :meth:`from_codes`."""
        if packed.dim() != 2 or packed.dtype is not torch.uint8:
            raise ValueError("Q4Weight: packed codes are (d_out, ceil(d_in / 2)) uint8")
        d_in = 2 * packed.shape[1] if d_in is None else int(d_in)
        if (d_in + 1) // 2 != packed.shape[1]:
            raise ValueError("Q4Weight: packed codes are (d_out, ceil(d_in / 2)) uint8")
        q = torch.stack([packed & 15, packed >> 4], 2).view(packed.shape[0], -1)[:, :d_in]
        return cls._lay_out(q, scale, center, group)

    @classmethod
    def from_codes(cls, codes, scale, center=None, group=64):
        """From codes (d_out, d_in) of an integer type, from 0 to 15, and scale and
        center (or None) (d_out, ceil(d_in / group))."""
        if codes.dtype.is_floating_point or codes.dtype is torch.bool or codes.dtype.is_complex:
            raise TypeError("Q4Weight: codes are integers")
        if codes.numel() and not 0 <= int(codes.min()) <= int(codes.max()) <= 15:
            raise ValueError("Q4Weight: codes are from 0 to 15")
        return cls._lay_out(codes.to(torch.uint8), scale, center, group)

    @classmethod
    def _lay_out(cls, q, scale, center, group):
        cls._check(q.shape, group)
        d_out, d_in = q.shape
        want = (d_out, -(-d_in // group))
        for t in (scale, center):
            if t is not None and (t.shape != want or not t.dtype.is_floating_point
                                  or t.device != q.device):
                raise ValueError("Q4Weight: scale and center are (d_out, ceil(d_in / group)) "
                                 "floats on the codes' device")
        unit = max(group, 64)
        tiles, cols = -(-d_out // 16), -(-d_in // unit) * unit
        full = q.new_full((tiles * 16, cols), 8)
        full[:d_out, :d_in] = q
        # output 8 h + l / 4, column 64 b + 32 (j / 2) + 8 (l % 4) + 4 (j % 2) + 2 v + e
        q = full.view(tiles, 2, 8, cols // 64, 2, 4, 2, 2, 2).permute(0, 3, 2, 5, 4, 6, 8, 7, 1)
        codes = (q[..., 0] | q[..., 1] << 4).flatten(6).view(torch.int32).view(tiles, -1, 32, 4)
        parts = []
        for t in (scale, center):
            if t is not None:
                p = torch.zeros(tiles * 16, cols // group, dtype=torch.bfloat16, device=q.device)
                p[:d_out, :want[1]] = t.detach()
                parts.append(p.view(tiles, 2, 8, cols // group).permute(0, 3, 2, 1))
        scales = torch.stack(parts, 4) if center is not None else parts[0]
        return cls(codes, scales.contiguous(), d_out, d_in, group, center is not None)

    def dequantize(self, dtype=torch.float32):
        """The weight (d_out, d_in) that the codes stand for."""
        tiles, groups = self.scales.shape[:2]
        cols = groups * self.group
        b = self.codes.view(torch.uint8).view(tiles, cols // 64, 8, 4, 2, 2, 2, 2)
        q = torch.stack([b & 15, b >> 4], 8).permute(0, 8, 2, 1, 4, 3, 5, 7, 6)
        q = q.reshape(tiles * 16, groups, self.group).float() - 8
        s = self.scales.float()
        if not self.has_center:
            s = s.unsqueeze(4)
        s = s.permute(4, 0, 3, 2, 1).reshape(-1, tiles * 16, groups, 1)
        w = q * s[0]
        if self.has_center:
            w += s[1]
        return w.view(tiles * 16, cols)[:self.d_out, :self.d_in].to(dtype)


def _rows(t, what, shape, dtype):
    """A tensor that the kernel reads or writes in place, by rows."""
    if t.shape != shape or t.dtype is not dtype or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"m3_rows_linear_q4: {what} is {tuple(shape)} with contiguous rows, of x's "
                         "element type")
    return t.stride(0) if shape[0] > 1 else max(t.stride(0), shape[1])


def m3_rows_linear_q4(x, weight, bias=None, norm_weight=None, eps=0.0, residual=None, split=None,
                      silu=False, out0=None, out1=None, overlap=False):
    """``act(residual + (bias + norm(x) @ weight.T))`` in one launch, with a
    :class:`Q4Weight`; x (rows, d_in) float32 or bfloat16, 1 to 8 rows.

    ``norm_weight`` (d_in,): apply the RMS norm x * rsqrt(mean(x^2) + eps) * w
    first (in float32, not rounded).  Columns [0, split) are returned in ``out0``
    (silu applied when ``silu``) and [split, d_out) in ``out1``; ``split`` defaults
    to d_out.  ``residual`` (rows, d_out) is added last and may be passed as
    ``out0`` to update it in place.  Returns (out0, out1), of x's element type; one
    without columns is None.  ``overlap``: launch as a programmatic dependent
    launch, which reads the first codes and scales before the kernel ahead of it on
    the stream completes (only when no queued kernel writes them).  A group's codes
    and inputs are summed before its scale and center come in: a row with an infinity,
    or past 1e35, may give NaN where its weights as floats give an infinity or a
    number; other rows do not change.  Inference only."""
    name = "m3_rows_linear_q4"
    if not isinstance(weight, Q4Weight):
        raise TypeError(f"{name}: weight is a Q4Weight")
    n, k = weight.d_out, weight.d_in
    shape, ty = x.shape, x.dtype
    if len(shape) != 2 or shape[1] != k or shape[0] > MAX_ROWS:
        raise ValueError(f"{name}: x is (rows, d_in) with at most {MAX_ROWS} rows and the weight's "
                         f"d_in")
    if H.needs_grad(x, bias, norm_weight, residual, out0, out1):
        raise ValueError(f"{name} has no derivative: call it under torch.no_grad()")
    code = H.code(ty)
    if (bias is not None and bias.shape != (n,)) or \
            (norm_weight is not None and norm_weight.shape != (k,)):
        raise ValueError(f"{name}: bias is (d_out,) and norm_weight (d_in,)")
    eps = float(eps)
    if not eps >= 0:
        raise ValueError(f"{name}: eps must not be negative")
    split = n if split is None else int(split)
    if not 0 <= split <= n:
        raise ValueError(f"{name}: split lies between 0 and d_out")
    H.refuse_tangents(name, x, bias, norm_weight, residual, out0, out1)
    dev = H.device_index(x, weight.codes, weight.scales, bias, norm_weight, residual, out0, out1)
    rows, rest = shape[0], n - split
    l0, l1, lr = split, rest, 0
    given = [t for t in (out0, out1) if t is not None]
    if out0 is not None:
        l0 = _rows(out0, "out0", (rows, split), ty)
    elif split:
        out0 = x.new_empty(rows, split)
    if out1 is not None:
        l1 = _rows(out1, "out1", (rows, rest), ty)
    elif rest:
        out1 = x.new_empty(rows, rest)
    if residual is not None:
        lr = _rows(residual, "residual", (rows, n), ty)
    if rows == 0:
        return out0, out1
    x2, lx = H.rows(x)
    b, nw = H.f32(bias), H.f32(norm_weight)
    H.launch(dev, _lib.load().m3_rows_linear_q4,
             RowsQ4Desc(rows, k, n, weight.group, weight.has_center, code, split, bool(silu), eps),
             x2.data_ptr(), lx, H.ptr(nw), weight.codes.data_ptr(),
             weight.scales.data_ptr(), H.ptr(b),
             H.ptr(residual), lr, H.ptr(out0), l0, H.ptr(out1), l1, bool(overlap))
    if given:
        increment_version(given)    # a backward pass that has saved one raises
    return out0, out1
