"""What the operators of a gated recurrent layer refuse on the host, before any
launch, and what their backward passes do with tensors that hooks give back."""

import contextlib
import ctypes

import pytest
import torch
from torch.autograd import forward_ad
from torch.autograd.graph import save_on_cpu, saved_tensors_hooks

from redpanda_b200 import _launch as H
from redpanda_b200 import _lib
from redpanda_b200 import gated as G
from redpanda_b200 import norm as N
from redpanda_b200 import quant as Q

z = torch.zeros


@pytest.mark.parametrize("call", [
    lambda: N.m3_add_rms_norm(z(2, 8), z(2, 8), z(7)),
    lambda: N.m3_add_rms_norm(z(2, 8), z(1, 8), z(8)),
    lambda: N.m3_add_rms_norm(z(2, 0), z(2, 0), z(0)),
    lambda: N.m3_add_rms_norm(z(2, 8), z(2, 8), z(8), eps=-1.0),
    lambda: N.m3_add_rms_norm(z(2, 8), z(2, 8), z(8), eps=float("nan")),
    lambda: N.m3_add_rms_norm(z(1, 40000), z(1, 40000), z(40000)),
    lambda: N.m3_rms_norm_8bit(z(2, 8), z(7)),
    lambda: N.m3_rms_norm_8bit(z(2, 8), z(8), residual=z(2, 7)),
    lambda: N.m3_rms_norm_8bit(z(2, 8), z(8), group=32),
    lambda: N.m3_rms_norm_8bit(z(2, 96), z(96), group=64),
    lambda: N.m3_rms_norm_8bit(z(2, 96), z(96), group=16),
    lambda: N.m3_rms_norm_8bit(z(2, 96), z(96), group=0),
    lambda: N.m3_rms_norm_8bit(z(2, 8), z(8, requires_grad=True)),
    lambda: G.m3_gated_scan(z(4, 8), z(4, 8), z(4, 8), z(8)),
    lambda: G.m3_gated_scan(z(1, 4, 8), z(1, 4, 7), z(1, 4, 8), z(8)),
    lambda: G.m3_gated_scan(z(1, 4, 8), z(1, 4, 8), z(1, 3, 8), z(8)),
    lambda: G.m3_gated_scan(z(1, 4, 8), z(1, 4, 8), z(1, 4, 8), z(7)),
    lambda: G.m3_gated_scan(z(1, 4, 0), z(1, 4, 0), z(1, 4, 0), z(0)),
    lambda: G.m3_gated_scan(*3 * [z(1, 4, 8)], z(8), c=0.0),
    lambda: G.m3_gated_scan(*3 * [z(1, 4, 8)], z(8), c=-1.0),
    lambda: G.m3_gated_scan(*3 * [z(1, 4, 8)], z(8), c=float("inf")),
    lambda: G.m3_gated_scan(*3 * [z(1, 4, 8)], z(8), c=float("nan")),
    lambda: G.m3_gated_scan(*3 * [z(1, 4, 8)], z(8), state=z(1, 7)),
    lambda: G.m3_gated_scan(*3 * [z(1, 4, 8)], z(8), state=z(1, 8, requires_grad=True)),
    lambda: G.m3_gated_scan(*3 * [z(1, 4, 8)], z(8), lengths=z(2, dtype=torch.int32)),
    lambda: G.m3_gated_scan(*3 * [z(1, 4, 8)], z(8), lengths=z(1)),
    lambda: G.m3_gated_scan(*3 * [z(1, 1, 1).expand(1, 2 ** 32 + 5, 1)], z(1)),
    lambda: G.m3_gated_step_(z(1, 7), *3 * [z(1, 8)], z(8)),
    lambda: G.m3_gated_step_(z(1, 8).double(), *3 * [z(1, 8)], z(8)),
    lambda: G.m3_gated_step_(z(8, 2).t(), *3 * [z(2, 8)], z(8)),
    lambda: G.m3_gated_step_(z(1, 8), z(1, 8, requires_grad=True), z(1, 8), z(1, 8), z(8)),
    lambda: G.m3_gated_step_(z(1, 8), *3 * [z(1, 1, 8)], z(8)),
])
def test_bad_arguments_raise_value_errors(call):
    with pytest.raises(ValueError):
        call()


@pytest.mark.parametrize("call", [
    lambda: N.m3_add_rms_norm(z(2, 8).half(), z(2, 8), z(8)),
    lambda: N.m3_add_rms_norm(z(2, 8), z(2, 8).double(), z(8)),
    lambda: N.m3_add_rms_norm(z(2, 8), z(2, 8), z(8), out_dtype=torch.float16),
    lambda: N.m3_rms_norm_8bit(z(2, 8), z(8), dtype=torch.uint8),
    lambda: N.m3_rms_norm_8bit(z(2, 8).half(), z(8)),
    lambda: G.m3_gated_scan(z(1, 4, 8).half(), z(1, 4, 8), z(1, 4, 8), z(8)),
])
def test_other_element_types_are_refused(call):
    with pytest.raises(TypeError):
        call()


CALLS = {
    "m3_add_rms_norm": (N.m3_add_rms_norm, lambda: [z(2, 8), z(2, 8), z(8)]),
    "m3_rms_norm_8bit": (N.m3_rms_norm_8bit, lambda: [z(2, 8), z(8), z(2, 8)]),
    "m3_gated_scan": (G.m3_gated_scan, lambda: [z(1, 4, 8), z(1, 4, 8), z(1, 4, 8), z(8)]),
    "m3_gated_scan_with_state": (G.m3_gated_scan_with_state, lambda: [
        z(1, 4, 8), z(1, 4, 8), z(1, 4, 8), z(8)]),
    "m3_gated_step_": (G.m3_gated_step_, lambda: [z(1, 8), z(1, 8), z(1, 8), z(1, 8), z(8)]),
    "m3_rows_linear_q4": (
        lambda x, b, n, r: Q.m3_rows_linear_q4(x, Q.Q4Weight.quantize(torch.ones(6, 40)), b, n,
                                               residual=r),
        lambda: [z(2, 40), z(6), z(40), z(2, 6)]),
}


@pytest.mark.parametrize("name", CALLS)
def test_cpu_tensors_and_forward_mode_tangents_are_refused(name):
    fn, make = CALLS[name]
    with pytest.raises(RuntimeError, match="CUDA"):
        fn(*make())
    for i in range(len(make())):
        with forward_ad.dual_level():
            a = make()
            a[i] = forward_ad.make_dual(a[i], torch.ones_like(a[i]))
            with pytest.raises(ValueError, match="forward-mode"):
                fn(*a)
            with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
                fn(*a)


class _Sizes:
    def __getattr__(self, name):
        def f(*a):
            return 64
        f.__name__ = name
        return f


@pytest.fixture
def launches(monkeypatch):
    seen = []
    monkeypatch.setattr(H, "device_index", lambda *ts: 0)
    monkeypatch.setattr(H, "on_device", lambda i: contextlib.nullcontext())
    monkeypatch.setattr(H, "launch", lambda i, *a: seen.append(a))
    monkeypatch.setattr(_lib, "load", lambda: _Sizes())
    return seen


def _calls(r):
    """Calls on strided views, and the leaves behind them."""
    base, w, res = r(3, 20, 24), r(8), r(3, 20, 8)
    leaves = [t.requires_grad_(True) for t in (base, w, res)]
    x, a, b = base[..., :8], base[..., 8:16], base[..., 16:]
    return leaves, {"add_norm": lambda: sum(N.m3_add_rms_norm(x, res, w)),
                    "gated": lambda: G.m3_gated_scan(x, a, b, w)}


def _strides(args):
    if args[0].__name__ == "m3_gated_bwd":
        return args[2].ld_x, args[2].ld_r, args[2].ld_i
    return (args[3],)


@pytest.mark.parametrize("name", ["add_norm", "gated"])
@pytest.mark.parametrize("unpack", [lambda t: t, lambda t: t.double(), lambda t: t.half(),
                                    lambda t: t[:1],
                                    lambda t: t.reshape(-1)[:1].expand(t.shape)])
def test_tensors_that_hooks_give_back(name, unpack, launches):
    """Another element type or shape raises before any launch; another layout is
    looked at again."""
    leaves, calls = _calls(lambda *s: torch.ones(*s))
    pack = lambda t: t.clone(memory_format=torch.contiguous_format)  # noqa: E731
    with saved_tensors_hooks(pack, unpack):
        y = calls[name]()
    launches.clear()
    same = unpack(torch.ones(2, 3))
    if same.dtype is torch.float32 and same.shape == (2, 3):
        y.sum().backward()
        assert set(_strides(launches[0])) == {8}
    else:
        with pytest.raises(RuntimeError, match="hooks"):
            y.sum().backward()
        assert not launches


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float64])
def test_buffers_are_float32_whatever_the_default(dtype, launches, monkeypatch):
    made = []
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, **k: made.append(empty(*a, **k)) or made[-1])
    old = torch.get_default_dtype()
    torch.set_default_dtype(dtype)
    try:
        f32 = lambda *s: torch.ones(*s, dtype=torch.float32)  # noqa: E731
        for name in ("add_norm", "gated"):
            leaves, calls = _calls(f32)
            calls[name]().sum().backward()
        N.m3_rms_norm_8bit(f32(3, 64), f32(64), residual=f32(3, 64), group=32)
        G.m3_gated_scan_with_state(*3 * [f32(2, 9, 8)], f32(8))
    finally:
        torch.set_default_dtype(old)
    assert made and all(t.dtype in (torch.float32, torch.uint8, torch.float8_e4m3fn) for t in made)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["add_norm", "gated"])
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


def test_c_entries_validate_before_device_work():
    """Status codes of bad descriptors and pointers (no device is touched)."""
    lib = _lib.load()
    buf = ctypes.create_string_buffer(8192)
    p = (ctypes.addressof(buf) + 255) // 256 * 256     # host memory: never dereferenced
    a, b, c, n = p + 512, p + 1024, p + 1536, None
    big = (1 << 30) + 1

    def add(rows=2, d=8, tx=0, ts=0, ty=0, eps=1e-5, x=p, lx=8, r=a, lr=8, w=p, y=b, s=c):
        return lib.m3_add_norm_fwd(_lib.AddNormDesc(rows, d, tx, ts, ty, eps), x, lx, r, lr, w, y, s,
                                   n, n)
    assert [add(x=n), add(r=n), add(w=n), add(y=n), add(s=n)] == [1] * 5
    assert [add(rows=0), add(d=0), add(eps=-1.0), add(eps=float("nan")), add(lx=7),
            add(lr=7)] == [2] * 6
    assert [add(tx=2), add(ts=-1), add(ty=7)] == [3] * 3
    assert add(d=40000, lx=40000, lr=40000) == 4
    assert [add(x=p + 2), add(r=a + 1, ts=1), add(y=b + 2), add(s=c + 2)] == [5] * 4
    assert [add(y=p), add(y=a), add(y=c), add(s=a, lr=9), add(s=p, tx=1)] == [11] * 5

    def addb(d=8, tx=0, s=p, ls=8, w=p, st=p, gy=a, gs=n, ds=b, dx=n, dw=p, ws=p, nws=0):
        return lib.m3_add_norm_bwd(_lib.AddNormDesc(2, d, tx, 0, 0, 1e-5), s, ls, w, st, gy, gs, ds,
                                   dx, dw, ws, nws, n)
    assert [addb(s=n), addb(w=n), addb(st=n), addb(gy=n), addb(ds=n), addb(dw=n),
            addb(tx=1)] == [1] * 7
    assert [addb(ls=7), addb(dx=c), addb(gs=p + 1), addb(ds=p), addb(ds=a),
            addb(tx=1, dx=b)] == [2, 4, 5, 11, 11, 11]

    def n8(rows=2, d=64, g=32, tx=0, ts=0, eps=1e-5, x=p, lx=64, r=n, lr=0, w=p, q=a, sc=b, s=n):
        return lib.m3_norm8_fwd(_lib.Norm8Desc(rows, d, g, tx, ts, 1, eps), x, lx, r, lr, w, q, sc,
                                s, n)
    assert [n8(x=n), n8(w=n), n8(q=n), n8(sc=n), n8(r=p, lr=64)] == [1] * 5
    assert [n8(rows=0), n8(d=0), n8(g=16), n8(g=128), n8(g=-32), n8(eps=-1.0), n8(lx=63),
            n8(r=a, lr=63, s=c)] == [2] * 8
    assert [n8(tx=2), n8(g=0, d=40000, lx=40000)] == [3, 4]
    assert [n8(x=p + 4), n8(lx=66), n8(q=a + 1), n8(r=c, lr=66, s=c + 256), n8(g=0, x=p + 2)] == \
        [5] * 5
    assert [n8(q=p), n8(r=a, lr=64, s=c), n8(r=c, lr=68, s=c)] == [11] * 3

    def args(**kw):
        v = dict(x=p, ld_x=8, rg=p, ld_r=8, ig=p, ld_i=8, decay=p)
        return _lib.GatedArgs(**{**v, **kw})

    def gated(B=1, L=4, D=8, ty=0, cc=8.0, ar=None, y=a, h=n, ck=n):
        return lib.m3_gated_fwd(_lib.GatedDesc(B, L, D, ty, cc), ar or args(), y, h, ck, n)
    assert lib.m3_gated_fwd(n, args(), a, n, n, n) == 1
    assert [gated(B=0), gated(L=0), gated(D=0), gated(cc=0.0), gated(cc=float("inf")),
            gated(cc=float("nan"))] == [2] * 6
    wide = args(ld_x=2 ** 31, ld_r=2 ** 31, ld_i=2 ** 31)
    assert [gated(B=big), gated(L=big), gated(D=big, ar=wide)] == [2] * 3
    assert [gated(ty=2), gated(y=n), gated(ar=args(x=n)), gated(ar=args(decay=n)),
            gated(ar=args(ld_r=7)), gated(ar=args(ig=p + 2)), gated(ck=p + 4), gated(y=p),
            gated(ar=args(state=b), h=b)] == [3, 1, 1, 1, 2, 5, 5, 11, 11]

    def gatedb(g=a, ck=b, dx=c, dr=c, di=c, dd=b, ws=p, nws=0, ar=None):
        return lib.m3_gated_bwd(_lib.GatedDesc(1, 4, 8, 0, 8.0), ar or args(), g, ck, dx, dr, di, dd,
                                ws, nws, n)
    assert [gatedb(g=n), gatedb(ck=n), gatedb(dx=n), gatedb(dr=n), gatedb(di=n),
            gatedb(dd=n)] == [1] * 6
    assert [gatedb(g=a + 2), gatedb(dr=p), gatedb(di=a), gatedb(ar=args(ld_i=3))] == [5, 11, 11, 2]

    def step(L=1, ar=None, h=a, y=b):
        return lib.m3_gated_step(_lib.GatedDesc(1, L, 8, 0, 8.0), ar or args(), h, y, n)
    assert [step(L=2), step(h=n), step(y=n), step(ar=args(state=c)), step(ar=args(lengths=c)),
            step(h=a + 2), step(y=a), step(h=p), step(ar=args(ld_x=7))] == \
        [2, 1, 1, 4, 4, 5, 11, 11, 2]

    def q4(rows=2, k=40, m=6, g=64, ce=1, ty=0, split=6, eps=0.0, x=p, lx=40, nw=n, co=a, sc=b,
           bi=n, r=n, lr=0, o0=c, l0=6, o1=n, l1=0):
        return lib.m3_rows_linear_q4(_lib.RowsQ4Desc(rows, k, m, g, ce, ty, split, 0, eps), x, lx,
                                     nw, co, sc, bi, r, lr, o0, l0, o1, l1, 0, n)
    assert [q4(x=n), q4(co=n), q4(sc=n), q4(o0=n), q4(split=3)] == [1] * 5
    assert [q4(rows=0), q4(k=0), q4(m=0), q4(g=16), q4(split=-1), q4(split=7), q4(lx=39),
            q4(l0=5), q4(r=p, lr=5), q4(nw=p, eps=-1.0)] == [2] * 10
    assert [q4(ty=2), q4(rows=9), q4(k=70000, lx=70000)] == [3, 4, 4]
    assert [q4(x=p + 2), q4(co=a + 8), q4(sc=b + 4), q4(o0=c + 1), q4(bi=p + 1)] == [5] * 5
    assert [q4(o0=p + 16), q4(r=c, lr=7, o0=c), q4(r=c + 4, lr=6)] == [11] * 3


def test_checkpoint_floats():
    f = lambda B, L, D: _lib.load().m3_gated_ckpt_floats(  # noqa: E731
        _lib.GatedDesc(B, L, D, 0, 8.0))
    assert f(2, 1, 8) == 16 and f(2, 4, 8) == 16 and f(2, 9, 8) == 48 and f(1, 0, 8) == 0


@pytest.mark.parametrize("center", [0, 1])
def test_scales_of_4_bit_weights_start_at_16_bytes(center):
    """They are copied 16 bytes at a time."""
    lib = _lib.load()
    buf = ctypes.create_string_buffer(8192)
    p = (ctypes.addressof(buf) + 255) // 256 * 256     # host memory: never dereferenced
    for off in (2, 4, 8, 12):
        desc = _lib.RowsQ4Desc(2, 40, 6, 64, center, 0, 6, 0, 0.0)
        assert lib.m3_rows_linear_q4(desc, p, 40, None, p + 512, p + 1024 + off, None, None, 0,
                                     p + 2048, 6, None, 0, 0, None) == 5


@pytest.mark.parametrize("rows", [0, 2])
def test_outputs_given_to_the_4_bit_product_count_as_changed(rows, launches):
    """A backward pass that has saved one raises."""
    w = Q.Q4Weight.quantize(torch.ones(6, 40), 32)
    for given in ("out0", "out1", "residual"):
        leaf = torch.ones(rows, {"out0": 2, "out1": 4, "residual": 6}[given], requires_grad=True)
        buf = leaf * 1
        y = buf.square()
        args = {given: buf, "split": 2}
        if given == "residual":
            args = {"residual": buf, "out0": buf}
        with torch.no_grad():
            Q.m3_rows_linear_q4(z(rows, 40), w, **args)
        if rows:
            with pytest.raises(RuntimeError, match="modified by an inplace"):
                y.sum().backward()
        else:
            y.sum().backward()
    r = torch.ones(2, 6, requires_grad=True)      # one that is only read does not
    y = (r * 1).square()
    with torch.no_grad():
        Q.m3_rows_linear_q4(z(2, 40), w, residual=r)
    y.sum().backward()


@pytest.mark.parametrize("given", ["out0", "out1"])
def test_outputs_with_forward_mode_tangents_are_refused(given):
    """They would keep the tangent of what they held."""
    w = Q.Q4Weight.quantize(torch.ones(6, 40), 32)
    with forward_ad.dual_level():
        out = forward_ad.make_dual(z(2, 3), torch.ones(2, 3))
        with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
            Q.m3_rows_linear_q4(z(2, 40), w, split=3, **{given: out})


def test_c_entries_refuse_ranges_that_overlap():
    """An output that shares some of its bytes with an input or another output; only
    the places that the header names may be the same (no device is touched: a call
    that passes ends at the device, or there without one)."""
    lib = _lib.load()
    buf = ctypes.create_string_buffer(1 << 16)
    p = (ctypes.addressof(buf) + 255) // 256 * 256     # host memory: never dereferenced
    at = [p + 2048 * i for i in range(16)]             # arrays below hold up to 1024 bytes
    n = None

    def add(x=at[0], lx=64, r=at[1], lr=64, w=at[2], y=at[3], s=at[4], st=at[5], tx=0):
        return lib.m3_add_norm_fwd(_lib.AddNormDesc(4, 64, tx, 0, 0, 1e-5), x, lx, r, lr, w, y, s,
                                   st, n)
    assert [add(y=at[0] + 1020), add(y=at[1] - 1020), add(y=at[4] + 16), add(s=at[0] + 512),
            add(s=at[1] + 4), add(r=at[4] - 4), add(x=at[0] + 1020, s=at[0] + 2040),
            add(y=at[2] + 252), add(s=at[2]), add(st=at[3] + 1020), add(st=at[1]), add(st=at[2] + 8),
            # strided rows reach further, and in place needs whole rows of one type
            add(x=at[6], lx=1024, y=at[8]), add(s=at[1], lr=65), add(s=at[0], tx=1)] == [11] * 15

    def addb(s=at[0], w=at[1], st=at[2], gy=at[3], gs=at[4], ds=at[5], dx=n, dw=at[7], tx=0):
        return lib.m3_add_norm_bwd(_lib.AddNormDesc(4, 64, tx, 0, 0, 1e-5), s, 64, w, st, gy, gs, ds,
                                   dx, dw, n, 0, n)
    assert [addb(ds=at[0] + 4), addb(ds=at[3] - 8), addb(ds=at[4] + 8), addb(ds=at[1]),
            addb(dw=at[0] + 512), addb(dw=at[1]), addb(dw=at[5] + 1020), addb(ds=at[2]),
            addb(tx=1, dx=at[4] + 2), addb(tx=1, dx=at[5] + 512), addb(tx=1, dx=at[7] + 4)] == [11] * 11

    def n8(x=at[0], lx=64, r=n, lr=0, w=at[2], q=at[3], sc=at[4], s=n, g=32):
        return lib.m3_norm8_fwd(_lib.Norm8Desc(4, 64, g, 0, 0, 1, 1e-5), x, lx, r, lr, w, q, sc, s,
                                n)
    assert [n8(q=at[0] + 1020), n8(q=at[2] + 128), n8(sc=at[0] + 4), n8(sc=at[3] + 252),
            n8(r=at[1], lr=64, s=at[1] + 16), n8(r=at[1], lr=64, s=at[0] + 16),
            n8(r=at[1], lr=64, s=at[2] + 16), n8(r=at[1], lr=64, s=at[3] - 16),
            n8(r=at[1], lr=64, s=at[5], sc=at[5] + 1020)] == [11] * 9

    # 2 rows of 4 steps of 16 channels: 512 bytes, 128 of a state or of checkpoints
    def args(**kw):
        v = dict(x=at[0], ld_x=16, rg=at[1], ld_r=16, ig=at[2], ld_i=16, decay=at[3], state=at[4],
                 lengths=at[5])
        return _lib.GatedArgs(**{**v, **kw})

    def gated(y=at[6], h=at[7], ck=at[8], **kw):
        return lib.m3_gated_fwd(_lib.GatedDesc(2, 4, 16, 0, 8.0), args(**kw), y, h, ck, n)
    assert [gated(y=at[0] + 508), gated(y=at[1] + 4), gated(y=at[2] - 508), gated(y=at[3]),
            gated(y=at[4] + 64), gated(y=at[5]), gated(h=at[4] + 64), gated(h=at[0]),
            gated(h=at[6] + 508), gated(ck=at[6]), gated(ck=at[7] + 64), gated(ck=at[4] + 8),
            gated(ck=at[3]), gated(x=at[9], ld_x=160, y=at[11])] == [11] * 14

    def gatedb(g=at[6], ck=at[7], dx=at[8], dr=at[9], di=at[10], dd=at[11], **kw):
        return lib.m3_gated_bwd(_lib.GatedDesc(2, 4, 16, 0, 8.0), args(state=n, **kw), g, ck, dx, dr,
                                di, dd, n, 0, n)
    assert [gatedb(dx=at[0] + 4), gatedb(dr=at[1] - 4), gatedb(di=at[2] + 508), gatedb(dx=at[6] + 4),
            gatedb(dr=at[7]), gatedb(dr=at[8]), gatedb(di=at[8] + 508), gatedb(di=at[9]),
            gatedb(dd=at[3]), gatedb(dd=at[10] + 4), gatedb(dd=at[7] + 64), gatedb(di=at[5]),
            gatedb(dx=at[3] + 4)] == [11] * 13

    def step(h=at[4], y=at[6], **kw):
        return lib.m3_gated_step(_lib.GatedDesc(2, 1, 16, 0, 8.0), args(state=n, lengths=n, **kw), h,
                                 y, n)
    assert [step(h=at[0] + 64), step(h=at[2] - 64), step(y=at[4] + 64), step(y=at[1] + 124),
            step(h=at[3] + 4), step(y=at[3])] == [11] * 6

    if not torch.cuda.is_available():                  # what may be the same
        assert {add(), add(s=at[1]), add(s=at[0]), add(s=at[1], x=at[1]), addb(), addb(gs=at[5]),
                addb(gs=n), n8(), n8(r=at[1], lr=64, s=at[1]), n8(r=at[1], lr=64, s=at[0]),
                gated(), gated(x=at[1], ig=at[1]), gated(state=n, h=n, ck=n), gatedb(),
                step()} == {9}


def test_outputs_of_the_4_bit_product_do_not_share_elements():
    """Halves of one buffer are two outputs; columns that both would write are refused
    (no device is touched: a call that passes ends there)."""
    lib = _lib.load()
    buf = ctypes.create_string_buffer(1 << 14)
    p = (ctypes.addressof(buf) + 255) // 256 * 256     # host memory: never dereferenced
    o = p + 4096

    def q4(o0, l0, o1, l1, split=4, rows=3, m=10):
        return lib.m3_rows_linear_q4(_lib.RowsQ4Desc(rows, 40, m, 64, 0, 0, split, 0, 0.0), p, 40,
                                     None, p + 1024, p + 2048, None, None, 0, o0, l0, o1, l1, 0, None)
    bad = [q4(o, 10, o, 10), q4(o, 10, o + 12, 10), q4(o + 8, 10, o, 10), q4(o, 10, o + 20, 10),
           q4(o, 10, o + 40, 10), q4(o, 10, o + 16, 11), q4(o, 4, o + 44, 6), q4(o, 9, o + 16, 9),
           q4(o, 10, o + 16, 10, rows=1, split=5)]
    assert bad == [11] * 9
    if not torch.cuda.is_available():
        good = {q4(o, 10, o + 16, 10), q4(o + 24, 10, o, 10), q4(o, 12, o + 16, 12),
                q4(o, 12, o + 24, 12), q4(o, 4, o + 48, 6), q4(o, 10, o + 16, 10, rows=1)}
        assert good == {9}
