"""The RMS norm with the residual's addition, and in 8 bits, against their
definition in 64 bits."""

import pytest
import torch

import seq_oracle as O
from redpanda_b200 import norm as N

pytestmark = pytest.mark.gpu
T = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-5


def inputs(rows, d, tx, ts, ty, seed):
    g = torch.Generator().manual_seed(seed)

    def n(*s, k=1.0):
        return torch.randn(*s, generator=g) * k
    return (n(rows, d, k=0.7).to(tx), (n(rows, d) + 0.3).to(ts), n(d, k=0.3) + 1,
            n(rows, d).to(ty), n(rows, d).to(ts))


def bounds(s, w, gy, gs, tx, ts, ty, k=96):
    """Reference (y, ds, dw) of the norm of s and what rounding allows: as the
    norm's own test, k = 96 roundings of e = 2^-24 on every path; the addition of
    gs is one of them."""
    rows = s.shape[0]
    y, dx, dw, _ = O.norm(s, w, None, EPS, True, gy)
    sd, g, wd = s.double(), gy.double(), w.double().abs()
    r = (sd.square().mean(1, keepdim=True) + EPS) ** -0.5
    mxh = sd.abs() * r
    q = g.abs() * wd
    mds = r * (q + mxh * (q * mxh).mean(1, keepdim=True)) + gs.double().abs()
    ds = dx + gs.double()
    return (y, k * O.E * mxh * wd + O.half_step(ty) * y.abs(),
            ds, k * O.E * mds + O.half_step(ts) * ds.abs(),
            k * O.E * mds + O.half_step(tx) * ds.abs(),
            dw, (k + rows) * O.E * (g.abs() * mxh).sum(0))


def near(got, ref, tol):
    assert ((got.detach().cpu().double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("tx,ts,ty", [(a, b, c) for a in T for b in T for c in T])
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 31), (700, 64), (9, 257), (5, 768), (33, 1000),
                                    (17, 1024), (6, 1030), (3, 4096), (2, 8200), (2, 16388),
                                    (1, 32767)])
def test_matches_definition(rows, d, tx, ts, ty):
    tx, ts, ty = T[tx], T[ts], T[ty]
    x, res, w, gy, gs = inputs(rows, d, tx, ts, ty, rows + 5 * d)
    leaves = [t.cuda().requires_grad_(True) for t in (x, res, w)]
    y, s = N.m3_add_rms_norm(*leaves, eps=EPS, out_dtype=ty)
    assert y.dtype == ty and s.dtype == ts
    # the stream's sum: fp32, rounded once
    assert torch.equal(s.detach().cpu(), (x.float() + res.float()).to(ts))
    dx, dres, dw = torch.autograd.grad((y, s), leaves, (gy.cuda(), gs.cuda()))
    assert dx.dtype == tx and dres.dtype == ts
    ry, ty_, rds, ts_, tx_, rdw, tw_ = bounds(s.detach().cpu(), w, gy, gs, tx, ts, ty)
    near(y, ry, ty_)
    near(dres, rds, ts_)
    near(dx, rds, tx_)
    near(dw, rdw, tw_)
    with torch.no_grad():   # the inference call gives the same bits
        y2, s2 = N.m3_add_rms_norm(*leaves, eps=EPS, out_dtype=ty)
    assert torch.equal(y, y2) and torch.equal(s, s2)


def test_one_gradient_alone():
    """y or s without a gradient: the other's alone, and zero for a weight that
    nothing depends on."""
    x, res, w, gy, gs = inputs(11, 96, torch.float32, torch.float32, torch.float32, 3)
    leaves = [t.cuda().requires_grad_(True) for t in (x, res, w)]
    y, s = N.m3_add_rms_norm(*leaves)
    zero = torch.zeros_like(gs)
    ref = bounds(s.detach().cpu(), w, gy, zero, *[torch.float32] * 3)
    dx, dres, dw = torch.autograd.grad(y, leaves, gy.cuda(), retain_graph=True)
    near(dx, ref[2], ref[3])
    near(dres, ref[2], ref[3])
    near(dw, ref[5], ref[6])
    dx, dres, dw = torch.autograd.grad(s, leaves, gs.cuda(), allow_unused=True)
    assert torch.equal(dx.cpu(), gs) and torch.equal(dres.cpu(), gs)
    assert dw is None


def test_strides_leading_dimensions_and_broadcast_gradient():
    g = torch.Generator().manual_seed(1)
    base, res = torch.randn(4, 6, 200, generator=g), torch.randn(4, 6, 72, generator=g)
    w = torch.randn(72, generator=g)
    for off in (0, 3, 64):          # 3: rows that no vector load can start at
        view = base.cuda()[..., off:off + 72]
        y, s = N.m3_add_rms_norm(view, res.cuda(), w.cuda())
        assert y.shape == s.shape == (4, 6, 72)
        assert torch.equal(s.cpu(), base[..., off:off + 72] + res)
        near(y, O.norm(s.cpu().view(24, 72), w, None, EPS, True).view(4, 6, 72),
             96 * O.E * 72 ** 0.5 * w.abs().max().double())
    # one residual row for all: its gradient is the sum over the rows
    x, one = base[0, :, :72], res[0, :1]
    up = torch.randn(6, 72, generator=g)
    a, b = x.cuda().requires_grad_(True), one.cuda().requires_grad_(True)
    y, s = N.m3_add_rms_norm(a, b.expand(6, 72), w.cuda())
    dx, dres = torch.autograd.grad(y, (a, b), up.cuda())
    assert dres.shape == (1, 72)
    total, mag = dx.double().sum(0, keepdim=True), dx.double().abs().sum(0, keepdim=True)
    assert ((dres.double() - total).abs() <= 8 * O.E * mag).all()


def test_gradient_against_differences():
    x, res, w, gy, gs = inputs(5, 48, *[torch.float32] * 3, 9)
    leaves = [t.cuda().requires_grad_(True) for t in (x, res, w)]
    grads = torch.autograd.grad(N.m3_add_rms_norm(*leaves, eps=EPS), leaves, (gy.cuda(), gs.cuda()))

    def value(a, b, c):
        s = a + b
        return (O.norm(s, c, None, EPS, True) * gy.double()).sum() + (s * gs.double()).sum()
    gen = torch.Generator().manual_seed(2)
    for i in range(3):
        v = torch.randn(leaves[i].shape, generator=gen).double()
        args, h = [x.double(), res.double(), w.double()], 1e-4
        f = []
        for sign in (1, -1):
            moved = list(args)
            moved[i] = moved[i] + sign * h * v
            f.append(value(*moved))
        diff = ((f[0] - f[1]) / (2 * h)).item()
        ours = grads[i].cpu().double() * v
        # differences: h^2 of a smooth function; the gradient: 96 e of its paths
        assert abs(ours.sum().item() - diff) <= 1e-5 * ours.abs().sum().item()


def test_empty_rows_and_refusals():
    w = torch.ones(8, device="cuda", requires_grad=True)
    x = torch.zeros(0, 8, device="cuda", requires_grad=True)
    y, s = N.m3_add_rms_norm(x, x, w)
    dx, dw = torch.autograd.grad(y.sum() + s.sum(), (x, w))
    assert dx.shape == (0, 8) and not dw.any()
    q, scale = N.m3_rms_norm_8bit(x.detach(), w.detach())
    assert q.shape == (0, 8) and scale.shape == (0, 1)
    with pytest.raises(RuntimeError, match="one device|CUDA"):
        N.m3_add_rms_norm(torch.zeros(2, 8, device="cuda"), torch.zeros(2, 8), w)
    with pytest.raises(ValueError, match="no_grad"):
        N.m3_rms_norm_8bit(torch.zeros(2, 8, device="cuda"), w)


def test_another_stream_and_capture():
    x, res, w, gy, gs = (t.cuda() for t in inputs(3000, 96, *[torch.float32] * 3, 4))

    def once():
        a = [t.detach().requires_grad_(True) for t in (x, res, w)]
        y, s = N.m3_add_rms_norm(*a)
        grads = torch.autograd.grad((y, s), a, (gy, gs))
        return (y.detach(), s.detach(), *grads, *(
            t.float() for t in N.m3_rms_norm_8bit(x, w, residual=res)))
    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = once()
    graph.replay()
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)


# ---------------------------------------------------------------- 8 bits

def check8(x, res, w, dtype, group, got):
    """y is off by 96 e of its size (the norm's bound); the scale by that at the
    group's largest and one division's rounding; q by half a step of the type (e4m3:
    2^-4 of the value, 2^-10 below 2^-6; int8: 1/2), and by y's error."""
    q, scale = got[0].cpu(), got[1].cpu().double()
    s = x
    if res is not None:
        s = (x.float() + res.float()).to(res.dtype)
        assert torch.equal(got[2].cpu(), s)
    y = O.norm(s.float(), w, None, EPS, True)
    top = 448.0 if dtype is torch.float8_e4m3fn else 127.0
    width = group or y.shape[1]
    parts = y.view(y.shape[0], -1, width)
    ref = (parts.abs().amax(-1) / top).clamp(min=2.0 ** -126)
    k = 98 * O.E
    assert ((scale - ref).abs() <= k * ref).all()
    back = q.double().view_as(parts) * scale[..., None]
    half = parts.abs() / 16 + scale[..., None] / 1024 if top == 448 else scale[..., None] / 2
    assert ((back - parts).abs() <= half * (1 + 1e-4) + 4 * k * parts.abs()).all()
    # a result of the definition, except where the quotient lies within rounding of a border
    lo, hi = ((parts / ref[..., None]) * (1 + f * 2 * k) for f in (-1, 1))
    rnd = (lambda v: v.float().clamp(-top, top).to(dtype).double()) if top == 448 else \
        (lambda v: v.round().clamp(-top, top))
    qd = q.double().view_as(parts)
    assert ((qd >= torch.minimum(rnd(lo), rnd(hi))) & (qd <= torch.maximum(rnd(lo), rnd(hi)))).all()


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("tx,ts", [("f32", None), ("bf16", None), ("f32", "f32"), ("bf16", "f32"),
                                   ("bf16", "bf16"), ("f32", "bf16")])
@pytest.mark.parametrize("rows,d,group", [(1, 1, None), (5, 77, None), (40, 64, 32), (9, 768, None),
                                          (9, 768, 128), (7, 992, 32), (3, 4096, 64), (3, 4097, None),
                                          (2, 8192, 128), (2, 9216, 32), (1, 32768, None)])
def test_8bit_matches_definition(rows, d, group, tx, ts, dtype):
    x, res, w, _, _ = inputs(rows, d, T[tx], T[ts or "f32"], torch.float32, rows + d)
    res = None if ts is None else res
    got = N.m3_rms_norm_8bit(x.cuda(), w.cuda(), residual=None if res is None else res.cuda(),
                             eps=EPS, dtype=dtype, group=group)
    assert got[0].dtype == dtype and got[0].shape == (rows, d)
    assert got[1].shape == (rows, d // group if group else 1)
    check8(x, res, w, dtype, group, got)


def test_8bit_of_strided_rows():
    g = torch.Generator().manual_seed(5)
    base, w = torch.randn(6, 300, generator=g), torch.randn(128, generator=g)
    for off in (0, 1, 4, 64):
        view = base[:, off:off + 128]
        for group in (None, 32):
            got = N.m3_rms_norm_8bit(base.cuda()[:, off:off + 128], w.cuda(), eps=EPS, group=group)
            check8(view, None, w, torch.float8_e4m3fn, group, got)


def test_8bit_of_zero_rows_tiny_rows_and_nan():
    x = torch.ones(5, 64)
    x[0] = 0
    x[1] *= 1e-30
    x[2, 40] = float("nan")
    x[4, :32] = 0
    w = torch.ones(64)
    w[3] = 0
    for dtype in (torch.float8_e4m3fn, torch.int8):
        q, scale = N.m3_rms_norm_8bit(x.cuda(), w.cuda(), dtype=dtype, group=32)
        q, scale = q.float().cpu(), scale.cpu()
        assert (scale[0] == 2.0 ** -126).all() and not q[0].any()
        assert torch.isfinite(q[1]).all() and torch.isfinite(scale[1]).all()
        assert torch.isnan(scale[2]).all()
        assert scale[4, 0] == 2.0 ** -126 and not q[4, :32].any() and q[4, 32:].all()
        assert torch.isfinite(scale[3]).all() and q[3, 3] == 0


def test_one_tensor_as_branch_and_stream():
    """x + x, whose gradient is the sum of both places'."""
    x, _, w, gy, gs = inputs(7, 200, *[torch.float32] * 3, 6)
    a, wc = x.cuda().requires_grad_(True), w.cuda()
    y, s = N.m3_add_rms_norm(a, a, wc)
    assert torch.equal(s.detach().cpu(), x + x)
    (da,) = torch.autograd.grad((y, s), (a,), (gy.cuda(), gs.cuda()))
    b = x.cuda().requires_grad_(True)
    c = x.cuda().requires_grad_(True)
    y, s = N.m3_add_rms_norm(b, c, wc)
    db, dc = torch.autograd.grad((y, s), (b, c), (gy.cuda(), gs.cuda()))
    assert torch.equal(da, db + dc)


def test_a_stream_changed_behind_the_call_raises_in_backward():
    """The sum is read again by the backward pass."""
    a = torch.randn(3, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda")
    y, s = N.m3_add_rms_norm(a, torch.zeros(3, 64, device="cuda"), w)
    with torch.no_grad():
        s.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_infinite_rows_are_nan_and_no_other():
    x = torch.randn(5, 300, generator=torch.Generator().manual_seed(3)).cuda()
    w = torch.ones(300, device="cuda")
    good = N.m3_add_rms_norm(x, x, w)[0]
    q0, s0 = N.m3_rms_norm_8bit(x, w)
    x[2, 7] = float("inf")
    y, _ = N.m3_add_rms_norm(x, x, w)
    q, sc = N.m3_rms_norm_8bit(x, w)
    keep = [0, 1, 3, 4]
    assert torch.isnan(y[2, 7]) and torch.equal(y[keep], good[keep])
    assert torch.isnan(sc[2]).all() and torch.equal(sc[keep], s0[keep])
    assert torch.equal(q[keep].view(torch.uint8), q0[keep].view(torch.uint8))


EVEN = [(5, 2), (7, 30), (300, 130), (9, 258), (9, 514), (9, 770), (5, 1022), (4, 1026), (3, 2050),
        (3, 5002), (2, 8194), (2, 16386), (1, 32766)]


@pytest.mark.parametrize("tx,ts,ty", [("f32", "f32", "f32"), ("bf16", "f32", "bf16"),
                                      ("bf16", "bf16", "bf16"), ("f32", "bf16", "f32")])
@pytest.mark.parametrize("rows,d", EVEN)
def test_rows_of_whole_pairs(rows, d, tx, ts, ty):
    test_matches_definition(rows, d, tx, ts, ty)


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("tx,ts", [("f32", None), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("rows,d", EVEN)
def test_8bit_rows_of_whole_pairs(rows, d, tx, ts, dtype):
    test_8bit_matches_definition(rows, d, None, tx, ts, dtype)


@pytest.mark.parametrize("rows,d", [(1, 8), (3, 257), (700, 64), (5000, 1000)])
def test_workspace_of_the_backward_is_what_it_uses(rows, d):
    """One partial of the weight gradient for each CTA (of four rows up to 256 columns,
    6 CTAs per SM there and 768 threads' worth further on); what lies behind stays as it
    was."""
    lib = N._lib.load()
    desc = N.AddNormDesc(rows, d, 0, 0, 0, EPS)
    n = lib.m3_add_norm_bwd_workspace_bytes(desc)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    ctas = min(-(-rows // 4) if d <= 256 else rows, 6 * sms if d <= 256 else
               sms * (768 // (-(-d // 256) * 32)))
    assert n == ctas * d * 4
    x, res, w, gy, gs = inputs(rows, d, *[torch.float32] * 3, rows)
    s, w, gy, gs = (x + res).cuda(), w.cuda(), gy.cuda(), gs.cuda()
    rstd = (s.square().mean(1) + EPS).rsqrt()
    ds, dw = torch.empty_like(s), torch.empty_like(w)
    ws = torch.full((n // 4 + 64,), 7.0, device="cuda")
    assert lib.m3_add_norm_bwd(desc, s.data_ptr(), d, w.data_ptr(), rstd.data_ptr(), gy.data_ptr(),
                               gs.data_ptr(), ds.data_ptr(), None, dw.data_ptr(), ws.data_ptr(), n,
                               torch.cuda.current_stream().cuda_stream) == 0
    _, _, rds, tol, _, rdw, tolw = bounds(s.cpu(), w.cpu(), gy.cpu(), gs.cpu(), *[torch.float32] * 3)
    near(ds, rds, tol)
    near(dw, rdw, tolw)
    assert (ws[n // 4:] == 7).all()
