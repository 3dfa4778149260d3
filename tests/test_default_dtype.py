"""Buffers of the sequence-model operators under another default element type of
torch's (``torch.set_default_dtype``): the kernels write float32 into them."""

import contextlib

import pytest
import torch

from redpanda_b200 import _launch as H
from redpanda_b200 import _lib
from redpanda_b200 import norm as N
from redpanda_b200 import selective as S
from redpanda_b200.sampling import m3_sample


@contextlib.contextmanager
def _default(dtype):
    old = torch.get_default_dtype()
    torch.set_default_dtype(dtype)
    try:
        yield
    finally:
        torch.set_default_dtype(old)


class _Sizes:
    """Stands for the library on the host: sizes, and entries that do nothing."""
    def __getattr__(self, name):
        return lambda *a: 64


def _f32(*shape):
    return torch.ones(*shape, dtype=torch.float32)


def _calls(r):
    x, w, b = r(2, 20, 8), r(8, 4), r(8)
    bc, A = r(2, 20, 4), r(8, 4)
    return [lambda g: N.m3_layer_norm(x.requires_grad_(g), b, b),
            lambda g: N.m3_rms_norm(x.requires_grad_(g), b),
            lambda g: S.m3_causal_conv_with_state(x.requires_grad_(g), w, b)[0],
            lambda g: S.m3_selective_scan_with_state(x.requires_grad_(g), x, A, bc, bc, D=b, z=x,
                                                     dt_bias=b)[0]]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float64])
def test_buffers_are_float32_whatever_the_default(dtype, monkeypatch):
    """Every buffer that the operators allocate on the way, forward and backward:
    float32 for float32 calls, or bytes whose number the library gave."""
    made = []
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, **k: made.append(empty(*a, **k)) or made[-1])
    monkeypatch.setattr(H, "device_index", lambda *ts: 0)
    monkeypatch.setattr(H, "on_device", lambda i: contextlib.nullcontext())
    monkeypatch.setattr(H, "launch", lambda *a: None)
    monkeypatch.setattr(_lib, "load", lambda: _Sizes())
    calls = _calls(_f32)
    with _default(dtype):
        for call in calls:
            with torch.no_grad():
                call(False)
            y = call(True)
            y.sum().backward()
    assert len(made) >= 8
    assert {t.dtype for t in made} <= {torch.float32, torch.uint8}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float64])
def test_results_are_the_same_under_another_default(dtype):
    def run():
        g = torch.Generator("cuda").manual_seed(4)
        r = lambda *s: torch.randn(*s, device="cuda", generator=g, dtype=torch.float32)  # noqa: E731
        out = []
        x, w, b, bc, A = r(2, 70, 8), r(8, 4), r(8), r(2, 70, 4), -r(8, 4).abs()
        for f in (lambda t: N.m3_layer_norm(t, b, b), lambda t: N.m3_rms_norm(t, b),
                  lambda t: S.m3_causal_conv(t, w, b),
                  lambda t: S.m3_selective_scan(t, x, A, bc, bc, D=b, z=x, dt_bias=b)):
            t = x.clone().requires_grad_(True)
            y = f(t)
            out += [y.detach(), *torch.autograd.grad(y, t, x)]
        out += S.m3_causal_conv_with_state(x, w, b)
        out += S.m3_selective_scan_with_state(x[:1].repeat(1, 9, 1), x[:1].repeat(1, 9, 1), A,
                                              bc[:1].repeat(1, 9, 1), bc[:1].repeat(1, 9, 1))
        out.append(S.m3_selective_step_(out[-1], x[:1, 0], x[:1, 0], A, bc[:1, 0], bc[:1, 0]))
        out.append(m3_sample(x[0], x[0, :, 0].sigmoid(), 0.7, 3, 0.9, 0.01))
        return out
    ref = run()
    with _default(dtype):
        got = run()
    for p, q in zip(ref, got):
        assert p.dtype == q.dtype and torch.equal(p, q)
