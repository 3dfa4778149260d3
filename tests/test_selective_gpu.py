"""Causal convolution and selective scan kernels against their definitions in
64 bits (seq_oracle), with bounds counted from the roundings."""

import pytest
import torch

import seq_oracle as O
from redpanda_b200 import selective as S

pytestmark = pytest.mark.gpu
T = {"f32": torch.float32, "bf16": torch.bfloat16}


def _rand(gen, *shape, lo=None, hi=None, scale=1.0, dtype=torch.float32):
    t = torch.rand(*shape, generator=gen) * (hi - lo) + lo if lo is not None \
        else torch.randn(*shape, generator=gen) * scale
    return t.to(dtype)


def _cuda(t):
    return None if t is None else t.cuda()


# ------------------------------------------------------------------ convolution

def _conv_inputs(B, L, D, K, dtype, ragged, state, seed):
    g = torch.Generator().manual_seed(seed)
    x = _rand(g, B, L, D, dtype=dtype)
    w, b = _rand(g, D, K, scale=0.5), _rand(g, D, scale=0.5)
    st = _rand(g, B, K - 1, D, dtype=dtype) if state else None
    n = torch.randint(0, L + 1, (B,), generator=g, dtype=torch.int32) if ragged else None
    if ragged:
        n[0], n[-1] = L, 0
    return x, w, b, st, n, _rand(g, B, L, D, dtype=dtype)


def _check_conv(x, w, b, st, n, gr, silu, y, so, dx, dw, db):
    B, L, D = x.shape
    K = w.shape[1]
    ry, rs, rdx, rdw, rdb = O.conv(x, w, b, silu, st, n, gr)
    bb = torch.zeros(D) if b is None else b
    absx = None if st is None else st.abs()
    mp = O.conv(x.abs(), w.abs(), bb.abs(), False, absx, n)[0]     # sum |w x| + |b|
    # p: K + 1 fused steps; silu: its slope is below 1.1, __expf's error
    # 2 + 1.2 |p| ulp (4 + 2.4 |p| half ulps), division and products 6 more
    k = K + 2
    tol = O.E * ((1.1 * k + 10 + 2.4 * mp) * mp) + O.half_step(x.dtype) * ry.abs()
    assert ((y.cpu().double() - ry).abs() <= tol).all()
    if so is not None:
        assert torch.equal(so.cpu().double(), rs)
    if dx is None:
        return
    # silu' is below 1.1 and its slope below 0.5; the same count on its paths
    c = O.E * (1.1 * (2 * K + 4) + 16 + (2.4 + 0.5 * k) * (1 + mp.max()))
    mag = O.conv(x.abs(), w.abs(), bb.abs(), False, absx, n, gr.abs().float())
    assert ((dx.cpu().double() - rdx).abs()
            <= 1.1 * c * mag[2] + O.half_step(x.dtype) * rdx.abs()).all()
    rows = B * L
    assert ((dw.cpu().double() - rdw).abs() <= (1.1 * c + rows * O.E) * mag[3]).all()
    if db is not None:
        assert ((db.cpu().double() - rdb).abs() <= (1.1 * c + rows * O.E) * mag[4]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,L,D,K,ragged,state,silu,bias", [
    (1, 1, 1, 1, False, False, True, True),
    (2, 1, 5, 4, False, True, True, True),
    (3, 2, 8, 4, True, True, True, True),
    (2, 37, 132, 4, True, False, True, True),
    (5, 65, 64, 2, True, True, False, True),
    (2, 33, 7, 3, False, True, True, False),
    (2, 40, 16, 8, True, True, True, True),
    (1, 130, 260, 4, False, False, True, True),
    (40, 9, 130, 5, True, True, False, False),
])
def test_conv_matches_definition(B, L, D, K, ragged, state, silu, bias, dtype):
    x, w, b, st, n, gr = _conv_inputs(B, L, D, K, T[dtype], ragged, state, B + L + D)
    b = b if bias else None
    xc, wc = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    bc = None if b is None else b.cuda().requires_grad_(True)
    y, so = S.m3_causal_conv_with_state(xc, wc, bc, silu, _cuda(st), _cuda(n))
    leaves = [t for t in (xc, wc, bc) if t is not None]
    gs = torch.autograd.grad(y, leaves, gr.cuda())
    _check_conv(x, w, b, st, n, gr, silu, y.detach(), so, gs[0], gs[1],
                gs[2] if bias else None)
    with torch.no_grad():
        assert torch.equal(y, S.m3_causal_conv(xc, wc, bc, silu, _cuda(st), _cuda(n)))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,off", [(64, 0), (64, 64), (30, 3)])
def test_conv_reads_strided_halves(D, off, dtype):
    g = torch.Generator().manual_seed(4)
    xz = _rand(g, 3, 21, 2 * D + 4, dtype=T[dtype]).cuda()
    x = xz[..., off:off + D]
    w, b = _rand(g, D, 4).cuda(), _rand(g, D).cuda()
    assert torch.equal(S.m3_causal_conv(x, w, b), S.m3_causal_conv(x.contiguous(), w, b))


def test_conv_ignores_what_lies_past_a_length():
    """NaN and infinities behind a row's length reach no output."""
    x, w, b, st, n, gr = _conv_inputs(4, 30, 64, 4, torch.float32, True, True, 8)
    bad, badg = x.clone(), gr.clone()
    for i in range(4):
        bad[i, n[i]:] = float("nan")
        badg[i, n[i]:] = float("inf")
    res = []
    for xx, gg in ((x, gr), (bad, badg)):
        xc, wc, bc = (t.cuda().requires_grad_(True) for t in (xx, w, b))
        y, so = S.m3_causal_conv_with_state(xc, wc, bc, True, st.cuda(), n.cuda())
        res.append((y.detach(), so, *torch.autograd.grad(y, (xc, wc, bc), gg.cuda())))
    for a, c in zip(*res):
        assert torch.equal(a, c)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("K", [1, 2, 4, 8])
def test_conv_parts_and_tokens_make_the_whole(K, dtype):
    """A sequence in two parts, and token by token, gives the bits of one call."""
    x, w, b, st, _, _ = _conv_inputs(3, 23, 36, K, T[dtype], False, True, 12)
    x, w, b, st = (t.cuda() for t in (x, w, b, st))
    y, so = S.m3_causal_conv_with_state(x, w, b, state=st)
    y1, s1 = S.m3_causal_conv_with_state(x[:, :9], w, b, state=st)
    y2, s2 = S.m3_causal_conv_with_state(x[:, 9:], w, b, state=s1)
    assert torch.equal(torch.cat([y1, y2], 1), y) and torch.equal(s2, so)
    cur = st.clone()
    for t in range(23):
        assert torch.equal(S.m3_causal_conv_step_(cur, x[:, t], w, b), y[:, t])
    assert torch.equal(cur, so)


def test_conv_gradient_against_differences():
    x, w, b, st, n, gr = _conv_inputs(3, 12, 6, 4, torch.float32, True, True, 31)
    xc, wc, bc = (t.cuda().requires_grad_(True) for t in (x, w, b))
    y = S.m3_causal_conv(xc, wc, bc, True, st.cuda(), n.cuda())
    grads = torch.autograd.grad(y, (xc, wc, bc), gr.cuda())
    gen = torch.Generator().manual_seed(32)
    for i, t in enumerate((x, w, b)):
        v = torch.randn(t.shape, generator=gen).double()
        f = []
        for s in (1, -1):
            a = [x.double(), w.double(), b.double()]
            a[i] = a[i] + s * 1e-4 * v
            f.append((O.conv(*a, True, st, n)[0] * gr.double()).sum().item())
        ours = (grads[i].cpu().double() * v)
        assert abs((f[0] - f[1]) / 2e-4 - ours.sum().item()) <= 1e-5 * ours.abs().sum().item()


# ------------------------------------------------------------------ scan

def _scan_inputs(B, L, D, N, dtype, ragged=False, state=False, gate=True, skip=True, bias=True,
                 seed=0, fast=False):
    g = torch.Generator().manual_seed(seed)
    a = dict(u=_rand(g, B, L, D, dtype=dtype), dt=_rand(g, B, L, D, scale=0.7, dtype=dtype),
             A=-_rand(g, D, N, lo=0.1, hi=float(N if not fast else 60)),
             Bm=_rand(g, B, L, N, dtype=dtype), Cm=_rand(g, B, L, N, dtype=dtype),
             D=_rand(g, D) if skip else None,
             z=_rand(g, B, L, D, dtype=dtype) if gate else None,
             dt_bias=_rand(g, D, lo=-5.0, hi=0.5) if bias else None,
             state=_rand(g, B, D, N) if state else None, lengths=None)
    if ragged:
        a["lengths"] = torch.randint(0, L + 1, (B,), generator=g, dtype=torch.int32)
        a["lengths"][0] = L
        if B > 1:
            a["lengths"][-1] = 0
    return a, _rand(g, B, L, D, dtype=dtype)


GRADS = dict(u="du", dt="ddt", A="dA", Bm="dB", Cm="dC", D="dD", z="dz", dt_bias="dbias")
NAMES = ("u", "dt", "A", "Bm", "Cm", "D", "z", "dt_bias")


def _run_scan(a, gr, softplus=True):
    c = {k: _cuda(v) for k, v in a.items()}
    for k in NAMES:
        if c[k] is not None:
            c[k].requires_grad_(True)
    y, h = S.m3_selective_scan_with_state(**c, softplus=softplus)
    leaves = [k for k in NAMES if c[k] is not None]
    gs = torch.autograd.grad(y, [c[k] for k in leaves], gr.cuda())
    return {"y": y.detach(), "h": h, **{GRADS[k]: v for k, v in zip(leaves, gs)}}


def _check_scan(a, gr, got, softplus=True):
    ref = O.scan(**a, g=gr, sp=softplus)
    mag = O.scan(**a, g=gr, sp=softplus, magnitude=True)
    B, L, D = a["u"].shape
    N = a["A"].shape[1]
    # roundings on a path: 10 per step there and back, N and D sums, the ends
    k = 20 * L + N + 64
    extra = dict(dA=B * L, dD=B * L, dbias=B * L, dB=D, dC=D)
    for name, v in got.items():
        r, m = ref[name], mag[name]
        tol = (k + extra.get(name, 0)) * O.E * m + O.half_step(v.dtype) * r.abs()
        off = (v.cpu().double() - r).abs()
        assert (off <= tol).all(), (name, (off - tol).max().item())
        # and in the norm: independent roundings add as their square root, so an
        # eighth of the worst case's count is generous
        scale = m.norm().item()
        assert off.norm().item() <= (k / 8 * O.E + O.half_step(v.dtype)) * scale, name


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,L,D,N,opt", [
    (1, 1, 1, 1, {}),
    (2, 1, 6, 4, dict(state=True)),
    (3, 15, 8, 8, dict(ragged=True)),
    (2, 16, 70, 16, dict(state=True, gate=False)),
    (3, 17, 64, 16, dict(ragged=True, state=True)),
    (2, 64, 128, 16, {}),
    (2, 50, 33, 24, dict(ragged=True)),
    (2, 40, 72, 32, dict(skip=False, bias=False)),
    (1, 35, 40, 64, dict(ragged=False, state=True)),
    (2, 20, 24, 128, dict(ragged=True, state=True)),
    (1, 33, 19, 65, dict(gate=False, skip=False)),
    (2, 130, 16, 3, dict(ragged=True, state=True)),
    (1, 200, 64, 16, dict(state=True)),          # split along time
    (3, 170, 40, 32, dict(ragged=True, state=True)),
    (1, 100, 64, 16, dict(fast=True)),           # gates that vanish within a step
])
def test_scan_matches_definition(B, L, D, N, opt, dtype):
    a, gr = _scan_inputs(B, L, D, N, T[dtype], seed=B * 100 + L + N, **opt)
    _check_scan(a, gr, _run_scan(a, gr))


def test_scan_step_size_without_softplus():
    a, gr = _scan_inputs(2, 33, 40, 16, torch.float32, seed=77)
    a["dt"] = a["dt"].abs() * 0.1
    a["dt_bias"] = a["dt_bias"].abs() * 0.01
    _check_scan(a, gr, _run_scan(a, gr, softplus=False), softplus=False)


def test_scan_softplus_past_its_threshold():
    a, gr = _scan_inputs(1, 20, 32, 8, torch.float32, seed=78)
    a["dt"] = a["dt"] * 15
    a["A"] = a["A"] * 0.02
    _check_scan(a, gr, _run_scan(a, gr))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_scan_split_along_time_equals_the_bound_and_batch(dtype):
    """A long prompt alone is split along time, in a batch it is not."""
    a, gr = _scan_inputs(1, 700, 64, 16, T[dtype], state=True, seed=5)
    one = {k: _cuda(v) for k, v in a.items()}
    y1, h1 = S.m3_selective_scan_with_state(**one)
    many = {k: (v if k in ("A", "D", "dt_bias") or v is None
                else v.expand(300, *v.shape[1:]).contiguous()) for k, v in one.items()}
    y2, h2 = S.m3_selective_scan_with_state(**many)
    mag = O.scan(**a, magnitude=True)
    k = 2 * (10 * 700 + 80)
    for p, q, m in ((y1, y2[:1], mag["y"]), (h1, h2[:1], mag["h"])):
        assert ((p.cpu().double() - q.cpu().double()).abs()
                <= k * O.E * m + 2 * O.half_step(p.dtype) * m).all()


def test_scan_reads_strided_views_and_mixed_types():
    g = torch.Generator().manual_seed(9)
    B, L, D, N = 2, 37, 64, 16
    xz = _rand(g, B, L, 2 * D).cuda()
    xd = _rand(g, B, L, 5 + 2 * N).cuda()
    A = -_rand(g, D, N, lo=0.5, hi=8.0).cuda()
    u, z, dt = xz[..., :D], xz[..., D:], _rand(g, B, L, D).cuda()
    Bm, Cm = xd[..., 5:5 + N], xd[..., 5 + N:]
    y = S.m3_selective_scan(u, dt, A, Bm, Cm, z=z)
    c = [t.contiguous() for t in (u, dt, Bm, Cm, z)]
    assert torch.equal(y, S.m3_selective_scan(c[0], c[1], A, c[2], c[3], z=c[4]))
    # activations of two types run in float32
    ub = u.to(torch.bfloat16)
    y2 = S.m3_selective_scan(ub, dt, A, Bm, Cm, z=z)
    assert y2.dtype == torch.float32
    assert torch.equal(y2, S.m3_selective_scan(ub.float(), dt, A, Bm, Cm, z=z))


def test_scan_ignores_what_lies_past_a_length():
    a, gr = _scan_inputs(4, 40, 32, 16, torch.float32, ragged=True, state=True, seed=21)
    bad, badg = {k: (None if v is None else v.clone()) for k, v in a.items()}, gr.clone()
    for i, n in enumerate(a["lengths"]):
        for k in ("u", "dt", "Bm", "Cm", "z"):
            bad[k][i, n:] = float("nan")
        badg[i, n:] = float("inf")
    p, q = _run_scan(a, gr), _run_scan(bad, badg)
    for k in p:
        assert torch.equal(p[k], q[k]), k
    assert torch.equal(p["h"][-1].cpu(), a["state"][-1])      # length 0: the state as given


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,D,N,opt", [(1, 5, 1, {}), (3, 64, 16, {}), (9, 40, 32, dict(gate=False)),
                                       (17, 33, 24, dict(skip=False, bias=False)),
                                       (2, 24, 128, {}), (8, 16, 64, {}), (5, 7, 6, {})])
def test_step_matches_definition(B, D, N, opt, dtype):
    a, _ = _scan_inputs(B, 1, D, N, T[dtype], state=True, seed=B + D + N, **opt)
    first = lambda t: None if t is None else t[:, 0]  # noqa: E731
    args = [first(a["u"]), first(a["dt"]), a["A"], first(a["Bm"]), first(a["Cm"])]
    kw = dict(D=a["D"], z=first(a["z"]), dt_bias=a["dt_bias"])
    h = a["state"].cuda()
    y = S.m3_selective_step_(h, *(_cuda(t) for t in args), **{k: _cuda(v) for k, v in kw.items()})
    ry, rh = O.token_step(a["state"], *args, **kw)
    my, mh = O.token_step(a["state"], *args, **kw, magnitude=True)
    k = 40 + N
    assert ((y.cpu().double() - ry).abs() <= k * O.E * my + O.half_step(y.dtype) * ry.abs()).all()
    assert ((h.cpu().double() - rh).abs() <= k * O.E * mh).all()


def test_tokens_after_a_prompt_continue_the_scan():
    """prompt (scan_with_state) + tokens (step) = one scan; a padded batch too."""
    a, _ = _scan_inputs(3, 30, 48, 16, torch.float32, seed=41)
    c = {k: _cuda(v) for k, v in a.items()}
    y, h = S.m3_selective_scan_with_state(**c)
    part = dict(c, **{k: c[k][:, :20] for k in ("u", "dt", "Bm", "Cm", "z")})
    _, hs = S.m3_selective_scan_with_state(**part)
    for t in range(20, 30):
        yt = S.m3_selective_step_(hs, c["u"][:, t], c["dt"][:, t], c["A"], c["Bm"][:, t],
                                  c["Cm"][:, t], D=c["D"], z=c["z"][:, t], dt_bias=c["dt_bias"])
        mag = O.scan(**a, magnitude=True)
        assert ((yt - y[:, t]).abs().cpu().double() <= 2 * (300 + 80) * O.E * mag["y"][:, t]).all()
    assert ((hs - h).abs().cpu().double() <= 2 * 380 * O.E * mag["h"]).all()


def test_scan_gradient_against_differences():
    a, gr = _scan_inputs(2, 18, 6, 8, torch.float32, ragged=True, state=True, seed=51)
    got = _run_scan(a, gr)
    gen = torch.Generator().manual_seed(52)
    for k in NAMES:
        v = torch.randn(a[k].shape, generator=gen).double()
        f = []
        for s in (1, -1):
            b = dict(a)
            b[k] = a[k].double() + s * 1e-4 * v
            f.append((O.scan(**b)["y"] * gr.double()).sum().item())
        ours = got[GRADS[k]].cpu().double() * v
        assert abs((f[0] - f[1]) / 2e-4 - ours.sum().item()) <= 3e-5 * ours.abs().sum().item(), k


def test_scan_shared_and_broadcast_inputs():
    """B = C one tensor, u expanded over the batch: gradients add up."""
    a, gr = _scan_inputs(3, 20, 32, 16, torch.float32, seed=61)
    u1, bc = a["u"][:1].cuda().requires_grad_(True), a["Bm"].cuda().requires_grad_(True)
    y = S.m3_selective_scan(u1.expand(3, 20, 32), a["dt"].cuda(), a["A"].cuda(), bc, bc)
    du, dbc = torch.autograd.grad(y, (u1, bc), gr.cuda())
    full = dict(u=a["u"][:1].expand(3, 20, 32), dt=a["dt"], A=a["A"], Bm=a["Bm"], Cm=a["Bm"])
    ref, mag = O.scan(**full, g=gr), O.scan(**full, g=gr, magnitude=True)
    k = 20 * 20 + 100
    assert ((du.cpu().double() - ref["du"].sum(0, keepdim=True)).abs()
            <= k * O.E * mag["du"].sum(0, keepdim=True)).all()
    assert ((dbc.cpu().double() - ref["dB"] - ref["dC"]).abs()
            <= k * O.E * (mag["dB"] + mag["dC"])).all()


@pytest.mark.parametrize("B,L", [(40, 33), (1, 300)])
def test_scan_is_deterministic_on_streams_and_in_graphs(B, L):
    a, gr = _scan_inputs(B, L, 64, 16, torch.float32, seed=71)
    c = {k: _cuda(v) for k, v in a.items()}
    gr = gr.cuda()

    def once():
        x = {k: (v if v is None or not v.is_floating_point() else v.detach().requires_grad_(True))
             for k, v in c.items() if k != "state"}
        y = S.m3_selective_scan(**x)
        return (y.detach(), *torch.autograd.grad(y, [x[k] for k in NAMES], gr))
    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        third = once()
    with torch.cuda.graph(g2):
        fourth = once()
    g1.replay()
    g2.replay()
    for p, q, r, s in zip(first, second, third, fourth):
        assert torch.equal(p, q) and torch.equal(p, r) and torch.equal(p, s)


def test_empty_batches_and_lengths():
    A = -torch.ones(8, 4, device="cuda")
    for B, L in ((0, 5), (3, 0)):
        u = torch.zeros(B, L, 8, device="cuda", requires_grad=True)
        bm = torch.zeros(B, L, 4, device="cuda")
        y, h = S.m3_selective_scan_with_state(u, u, A, bm, bm)
        assert y.shape == (B, L, 8) and h.shape == (B, 8, 4) and not h.any()
        assert torch.autograd.grad(y.sum(), u)[0].shape == u.shape
        w = torch.ones(8, 4, device="cuda", requires_grad=True)
        y, st = S.m3_causal_conv_with_state(u, w)
        assert st.shape == (B, 3, 8) and not torch.autograd.grad(y.sum(), w)[0].any()
    h = torch.zeros(0, 8, 4, device="cuda")
    e = torch.zeros(0, 8, device="cuda")
    assert S.m3_selective_step_(h, e, e, A, e[:, :4], e[:, :4]).shape == (0, 8)


def test_in_place_steps_refuse_autograd_and_loose_states():
    d = dict(device="cuda")
    A, e, b = -torch.ones(8, 4, **d), torch.zeros(2, 8, **d), torch.zeros(2, 4, **d)
    with pytest.raises(ValueError, match="no_grad"):
        S.m3_selective_step_(torch.zeros(2, 8, 4, **d), e.clone().requires_grad_(True), e, A, b, b)
    with pytest.raises(ValueError, match="contiguous"):
        S.m3_selective_step_(torch.zeros(2, 4, 8, **d).transpose(1, 2), e, e, A, b, b)
    with pytest.raises(ValueError, match="contiguous"):
        S.m3_causal_conv_step_(torch.zeros(2, 8, 3, **d).transpose(1, 2), e, torch.ones(8, 4, **d))
    with pytest.raises(ValueError, match="differentiable"):
        S.m3_selective_scan(e[:, None], e[:, None], A, b[:, None], b[:, None],
                            state=torch.zeros(2, 8, 4, **d, requires_grad=True))


def test_steps_of_size_zero_leave_the_state():
    """A gate of a step of size zero is one exactly, in the scan and the step
    (masked steps within a chunk rest on it)."""
    g = torch.Generator().manual_seed(91)
    B, L, D, N = 2, 100, 40, 16
    h0 = _rand(g, B, D, N).cuda()
    zero, b = torch.zeros(B, L, D, device="cuda"), _rand(g, B, L, N).cuda()
    A = -_rand(g, D, N, lo=0.1, hi=50.0).cuda()
    _, h = S.m3_selective_scan_with_state(zero, zero, A, b, b, softplus=False, state=h0)
    assert torch.equal(h, h0)
    h = h0.clone()
    S.m3_selective_step_(h, zero[:, 0], zero[:, 0], A, b[:, 0], b[:, 0], softplus=False)
    assert torch.equal(h, h0)


@pytest.mark.parametrize("kind", ["int64", "int16", "uint8", "far"])
def test_lengths_of_other_integer_types_and_out_of_range(kind):
    g = torch.Generator().manual_seed(92)
    x, w = _rand(g, 3, 20, 8).cuda(), _rand(g, 8, 4).cuda()
    n = torch.tensor([7, 20, 0])
    given = torch.tensor([7, 2 ** 40, -5]) if kind == "far" else n.to(getattr(torch, kind))
    ref = S.m3_causal_conv_with_state(x, w, lengths=n.to(torch.int32).cuda())
    got = S.m3_causal_conv_with_state(x, w, lengths=given.cuda())
    assert torch.equal(ref[0], got[0]) and torch.equal(ref[1], got[1])


def test_calls_side_by_side_on_two_streams():
    """Two scans and their backward passes at once: each has its own workspace."""
    a, gr = _scan_inputs(1, 400, 64, 16, torch.float32, seed=95)
    b, gb = _scan_inputs(1, 400, 64, 16, torch.float32, seed=96)
    ref = [_run_scan(a, gr), _run_scan(b, gb)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for s, (p, q) in zip(streams, ((a, gr), (b, gb))):
            with torch.cuda.stream(s):
                got.append(_run_scan(p, q))
        torch.cuda.synchronize()
        for r, o in zip(ref, got):
            assert all(torch.equal(r[k], o[k]) for k in r)


def test_double_backward_is_refused():
    a, gr = _scan_inputs(1, 20, 16, 8, torch.float32, seed=97)
    c = {k: _cuda(v) for k, v in a.items()}
    c["u"].requires_grad_(True)
    y = S.m3_selective_scan(**c)
    (du,) = torch.autograd.grad((y * y).sum(), c["u"], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(du.sum(), c["u"])


def _growing(seed):
    a, gr = _scan_inputs(1, 2000, 64, 16, torch.float32, gate=False, skip=False, bias=False,
                         seed=seed)
    a["A"] = a["A"].abs() / 160 + 0.95          # 0.95 to 1.05
    a["dt"] = torch.full_like(a["dt"], 4.0)
    return a, gr


def test_growth_over_empty_runs_keeps_zeros():
    """A > 0: a state that is zero over a long part stays zero there, although the
    part's whole growth is past float32; its gradient, from the back, too."""
    a, _ = _growing(51)
    a["u"][:, :-8] = 0
    with torch.no_grad():
        y, h = S.m3_selective_scan_with_state(**{k: _cuda(v) for k, v in a.items()},
                                              softplus=False)
    ref, mag = O.scan(**a, sp=False), O.scan(**a, sp=False, magnitude=True)
    # the 8 steps that are not empty: 10 roundings each, the sum over the states
    for got, k in ((y, "y"), (h, "h")):
        assert ((got.cpu().double() - ref[k]).abs() <= (20 * 8 + 16 + 64) * O.E * mag[k]).all()
    a, gr = _growing(52)
    a["u"].zero_()
    gr[:, 8:] = 0
    _check_scan(a, gr, _run_scan(a, gr, softplus=False), softplus=False)


@pytest.mark.parametrize("low", [-float("inf"), -3e38])
def test_gates_of_the_lowest_values_are_zero_up_to_the_length(low):
    """A column of A at the type's lowest values forgets at every step, and the
    state behind a length that ends inside a chunk is the one at the length."""
    a, _ = _scan_inputs(2, 13, 8, 4, torch.float32, seed=52)
    a["lengths"] = torch.tensor([13, 5], dtype=torch.int32)
    a["A"][:, 1] = low
    y, h = S.m3_selective_scan_with_state(**{k: _cuda(v) for k, v in a.items()})
    b = dict(a, A=a["A"].clone())
    b["A"][:, 1] = -1e6          # exp(-1e6 de) is 0 for every step size here
    y1, h1 = S.m3_selective_scan_with_state(**{k: _cuda(v) for k, v in b.items()})
    assert torch.equal(y, y1) and torch.equal(h, h1) and h.isfinite().all()
