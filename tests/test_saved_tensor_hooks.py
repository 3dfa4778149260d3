"""Backward passes of the operators when saved tensors come back through hooks
(``torch.autograd.graph.saved_tensors_hooks``): with another layout than the
strided views that the forward read, or as something else altogether."""

import contextlib

import pytest
import torch
from torch.autograd.graph import save_on_cpu, saved_tensors_hooks

from redpanda_b200 import _launch as H
from redpanda_b200 import _lib
from redpanda_b200 import norm as N
from redpanda_b200 import selective as S


class _Sizes:
    def __getattr__(self, name):
        def f(*a):
            return 64
        f.__name__ = name
        return f


def _calls(r):
    """Calls on strided views, and the leaves behind them."""
    base, w, b = r(3, 20, 24), r(8, 4), r(8)
    dt, bc, A = r(3, 20, 8), r(3, 20, 13), -r(8, 4).abs()
    leaves = [t.requires_grad_(True) for t in (base, w, b, dt, bc, A)]
    x, z, Bm, Cm = base[..., 8:16], base[..., 16:], bc[..., 1:5], bc[..., 7:11]
    return leaves, {
        "layer_norm": lambda: N.m3_layer_norm(x, b, b),
        "rms_norm": lambda: N.m3_rms_norm(x, b),
        "conv": lambda: S.m3_causal_conv(x, w, b),
        "scan": lambda: S.m3_selective_scan(x, dt, A, Bm, Cm, D=b, z=z, dt_bias=b),
    }


def _strides_of_launch(args):
    """Row strides that a launch of a backward pass was given."""
    fn = args[0].__name__
    if fn == "m3_selective_bwd":
        a = args[2]
        return {"u": a.u_ld, "dt": a.dt_ld, "z": a.z_ld, "B": a.B_ld, "C": a.C_ld}
    return {"x": args[3]}


WANT = {"layer_norm": dict(x=8), "rms_norm": dict(x=8), "conv": dict(x=8),
        "scan": dict(u=8, dt=8, z=8, B=4, C=4)}


@pytest.fixture
def launches(monkeypatch):
    seen = []
    monkeypatch.setattr(H, "device_index", lambda *ts: 0)
    monkeypatch.setattr(H, "on_device", lambda i: contextlib.nullcontext())
    monkeypatch.setattr(H, "launch", lambda i, *a: seen.append(a))
    monkeypatch.setattr(_lib, "load", lambda: _Sizes())
    return seen


@pytest.mark.parametrize("name", WANT)
def test_row_strides_are_those_of_the_unpacked_tensors(name, launches):
    leaves, calls = _calls(lambda *s: torch.ones(*s))
    pack = lambda t: t.clone(memory_format=torch.contiguous_format)  # noqa: E731
    with saved_tensors_hooks(pack, lambda t: t):
        y = calls[name]()
    launches.clear()
    y.sum().backward()
    assert len(launches) == 1 and _strides_of_launch(launches[0]) == WANT[name]
    # without hooks: the views' own
    y = calls[name]()
    launches.clear()
    y.sum().backward()
    got = _strides_of_launch(launches[0])
    assert got.get("x", got.get("u")) == 24 and got.get("B", 13) == 13


@pytest.mark.parametrize("unpack", [lambda t: t.double(), lambda t: t.half(), lambda t: t[:1],
                                    lambda t: t.reshape(-1)[:1].expand(t.shape)])
@pytest.mark.parametrize("name", WANT)
def test_other_tensors_are_refused_or_laid_out(name, unpack, launches):
    """Another element type or shape raises before any launch; an expanded tensor
    is laid out for the kernel."""
    leaves, calls = _calls(lambda *s: torch.ones(*s))
    with saved_tensors_hooks(lambda t: t, unpack):
        y = calls[name]()
    launches.clear()
    same = unpack(torch.ones(2, 3))
    if same.dtype is torch.float32 and same.shape == (2, 3):
        y.sum().backward()
        assert _strides_of_launch(launches[0]) == WANT[name]
    else:
        with pytest.raises(RuntimeError, match="hooks"):
            y.sum().backward()
        assert not launches


@pytest.mark.gpu
@pytest.mark.parametrize("name", WANT)
def test_gradients_with_tensors_saved_on_the_cpu(name):
    res = []
    for hooks in (contextlib.nullcontext(), save_on_cpu(), save_on_cpu(pin_memory=True)):
        g = torch.Generator("cuda").manual_seed(8)
        leaves, calls = _calls(lambda *s: torch.randn(*s, device="cuda", generator=g))
        with hooks:
            y = calls[name]()
        grads = torch.autograd.grad(y.square().sum(), leaves, allow_unused=True)
        res.append([y.detach(), *(t for t in grads if t is not None)])
    for other in res[1:]:
        assert all(torch.equal(p, q) for p, q in zip(res[0], other))


@pytest.mark.gpu
def test_tensors_left_on_the_cpu_are_refused():
    for name in WANT:
        leaves, calls = _calls(lambda *s: torch.randn(*s, device="cuda"))
        with saved_tensors_hooks(lambda t: t.cpu(), lambda t: t):
            y = calls[name]()
        with pytest.raises(RuntimeError, match="CUDA|one device"):
            y.sum().backward()
