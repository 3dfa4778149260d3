"""silu and its derivative on the operators over the whole range of their argument,
element by element (a sum would hide a small gate behind a large one).

Relative error: the exponent x log2(e) is rounded once and log2(e) itself is off by
0.23 e (e = 2^-24), so e^-x is off by 1.23 |x| e, beside ex2's 4 e, rcp's 2 e and
four more roundings of sums and products: (1.3 |x| + 10) e of silu, and of
s (1 + |x| (1 - s)) for silu' = s (1 + x (1 - s)), whose paths cancel near
x = -1.28, with two roundings more.  Where 1 + e^-x passes 2^126 its reciprocal is
flushed: below x = -87.3 the gate is 0, off by less than 88 * 2^-126."""

import pytest
import torch

from redpanda_b200 import selective as S

pytestmark = pytest.mark.gpu
E, FLUSH = 2.0 ** -24, 88 * 2.0 ** -126


def _arguments():
    g = torch.Generator().manual_seed(1)
    near = torch.randn(5000, generator=g) * 3
    wide = torch.rand(7000, generator=g) * 200 - 100
    return torch.cat([near, wide, torch.tensor([0.0, -0.0, -87.0, -88.5, -100.0, 100.0])])


def _reference(x):
    x = x.double()
    s = 1 / (1 + torch.exp(-x))
    return x * s, s * (1 + x * (1 - s)), s * (1 + x.abs() * (1 - s)), (1.3 * x.abs() + 10) * E


def test_convolution_activation_over_its_range():
    x = _arguments()
    y, dy, mag, rel = _reference(x)
    xc = x.cuda().view(1, 1, -1).requires_grad_(True)
    got = S.m3_causal_conv(xc, torch.ones(len(x), 1, device="cuda"))
    (dx,) = torch.autograd.grad(got.sum(), xc)
    assert ((got.detach().cpu().view(-1).double() - y).abs() <= rel * y.abs() + FLUSH).all()
    assert ((dx.cpu().view(-1).double() - dy).abs() <= (rel + 2 * E) * mag + FLUSH).all()
    step = S.m3_causal_conv_step_(torch.empty(1, 0, len(x), device="cuda"), xc.detach()[0],
                                  torch.ones(len(x), 1, device="cuda"))
    assert torch.equal(step[0], got[0, 0])


def test_scan_gate_over_its_range():
    """No state (B = 0): y = D u silu(z), dz = u silu'(z), with u = D = 1."""
    z = _arguments()
    y, dy, mag, rel = _reference(z)
    n = len(z)
    one, zero = torch.ones(1, 1, n, device="cuda"), torch.zeros(1, 1, 4, device="cuda")
    zc = z.cuda().view(1, 1, -1).requires_grad_(True)
    kw = dict(D=torch.ones(n, device="cuda"))
    A = -torch.ones(n, 4, device="cuda")
    got = S.m3_selective_scan(one, one, A, zero, zero, z=zc, **kw)
    (dz,) = torch.autograd.grad(got.sum(), zc)
    assert ((got.detach().cpu().view(-1).double() - y).abs() <= rel * y.abs() + FLUSH).all()
    assert ((dz.cpu().view(-1).double() - dy).abs() <= (rel + 2 * E) * mag + FLUSH).all()
    h = torch.zeros(1, n, 4, device="cuda")
    step = S.m3_selective_step_(h, one[0], one[0], A, zero[0], zero[0], z=zc.detach()[0], **kw)
    assert ((step.cpu().view(-1).double() - y).abs() <= rel * y.abs() + FLUSH).all()
