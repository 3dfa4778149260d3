"""Batches that the backward passes walk in several turns: a CTA (or warp) takes
more than two rows or runs, with a remainder, so that what it carries from one to
the next -- fetched inputs, sums of the parameters' gradients, the gradient of the
state -- is compared with the definition in 64 bits."""

import pytest
import torch

import seq_oracle as O
from redpanda_b200 import _lib
from redpanda_b200 import norm as N
from redpanda_b200 import selective as S
from test_norm_gpu import _check, _inputs
from test_selective_gpu import T, _check_scan, _run_scan, _scan_inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("tx,ty", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("rows,d", [(9001, 64), (9003, 61), (4001, 300), (5001, 1000), (2600, 1028),
                                    (400, 9000), (311, 16385)])
def test_norm_over_many_rows(rows, d, tx, ty, rms):
    tx, ty = T[tx], T[ty]
    desc = _lib.NormDesc(rows, d, 0, 0, rms, 1e-5)
    ctas = _lib.load().m3_norm_bwd_workspace_bytes(desc) // (8 * d)
    assert rows > 2 * ctas * (4 if d <= 256 else 1)
    x, w, b, g = _inputs(rows, d, tx, rows + d)
    g = g.to(ty)
    xc, wc, bc = (t.cuda().requires_grad_(True) for t in (x, w, b))
    if rms:
        y, b, db = N.m3_rms_norm(xc, wc, eps=1e-5, out_dtype=ty), None, None
        dx, dw = torch.autograd.grad(y, (xc, wc), g.cuda())
    else:
        y = N.m3_layer_norm(xc, wc, bc, eps=1e-5, out_dtype=ty)
        dx, dw, db = torch.autograd.grad(y, (xc, wc, bc), g.cuda())
    _check(x, w, b, g, 1e-5, rms, ty, y.detach(), dx, dw, db)


def _conv_reference(x, w, b, silu, state, n, g):
    """(y, state, dx, dw, db) in 64 bits, every row at once."""
    x, w, b, g = (t.double() for t in (x, w, b, g))
    B, L, D = x.shape
    K = w.shape[1]
    live = (torch.arange(L) < n[:, None])[..., None]
    x, g = torch.where(live, x, 0), torch.where(live, g, 0)
    past = torch.zeros(B, K - 1, D, dtype=torch.float64) if state is None else state.double()
    rows = torch.cat([past, x], 1)
    p = b + sum(rows[:, k:k + L] * w[:, k] for k in range(K))
    s = 1 / (1 + torch.exp(-p))
    y = torch.where(live, p * s if silu else p, 0)
    q = g * (s * (1 + p * (1 - s)) if silu else 1.0)
    qz = torch.cat([q, torch.zeros(B, K - 1, D, dtype=torch.float64)], 1)
    dx = torch.where(live, sum(qz[:, K - 1 - k:K - 1 - k + L] * w[:, k] for k in range(K)), 0)
    dw = torch.stack([(q * rows[:, k:k + L]).sum((0, 1)) for k in range(K)], 1)
    at = (n[:, None].long() + torch.arange(K - 1))[..., None].expand(B, K - 1, D)
    return y, rows.gather(1, at), dx, dw, q.sum((0, 1))


def test_conv_reference_is_the_definition():
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    for K, silu in ((4, True), (3, False), (1, True)):
        x, w, b, st, gr = r(3, 7, 5), r(5, K), r(5), r(3, K - 1, 5), r(3, 7, 5)
        n = torch.tensor([7, 0, 3])
        for p, q in zip(_conv_reference(x, w, b, silu, st, n, gr), O.conv(x, w, b, silu, st, n, gr)):
            # the same products in 64 bits, at most 21 of them added in another order
            assert ((p - q).abs() <= 1e-13 * (1 + q.abs())).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,L,D,K,silu", [(6000, 3, 12, 4, True), (110, 1700, 8, 4, True),
                                          (1001, 70, 132, 3, True), (901, 70, 130, 8, False),
                                          (700, 251, 13, 2, True)])
def test_conv_over_many_runs(B, L, D, K, silu, dtype):
    dt = T[dtype]
    desc = _lib.ConvDesc(B, L, D, K, 0, int(silu))
    workers = _lib.load().m3_causal_conv_bwd_workspace_bytes(desc) // (4 * (K + 1) * D)
    assert B * ((L + 31) // 32) > 2 * 8 * workers
    g = torch.Generator().manual_seed(B + L)
    r = lambda *s, c=1.0: torch.randn(*s, generator=g) * c  # noqa: E731
    x, w, b, st, gr = r(B, L, D).to(dt), r(D, K, c=0.5), r(D, c=0.5), r(B, K - 1, D).to(dt), \
        r(B, L, D).to(dt)
    n = torch.randint(0, L + 1, (B,), generator=g)
    n[::3], n[1::5] = L, 0
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    y, so = S.m3_causal_conv_with_state(*leaves, silu, st.cuda(), n.cuda())
    got = [y.detach(), so, *torch.autograd.grad(y, leaves, gr.cuda())]
    ry, rs, *rg = _conv_reference(x, w, b, silu, st, n, gr)
    ab = [t.abs() for t in (x, w, b)]
    my, _, *mg = _conv_reference(*ab, False, st.abs(), n, gr.abs())
    # the counts of the roundings are those of the small cases: K + 2 on p, silu's
    # slope below 1.1, its error 10 + 2.4 |p|; silu' the same on its paths
    k = K + 2
    half = O.half_step(dt)
    assert ((got[0].cpu().double() - ry).abs()
            <= O.E * (1.1 * k + 10 + 2.4 * my) * my + half * ry.abs()).all()
    assert torch.equal(got[1].cpu().double(), rs)
    c = 1.1 * O.E * (1.1 * (2 * K + 4) + 16 + (2.4 + 0.5 * k) * (1 + my.max()))
    assert ((got[2].cpu().double() - rg[0]).abs() <= c * mg[0] + half * rg[0].abs()).all()
    # a parameter's sum: the additions of a warp's runs (four at most here, 32 steps
    # each), of 8 warps and of the CTAs' partials
    adds = (4 * 32 + 8 + workers) * O.E
    for a, ref, m in zip(got[3:], rg[1:], mg[1:]):
        assert ((a.cpu().double() - ref).abs() <= (c + adds) * m).all()


def _scan_bgroups(B, L, D, Ns):
    """Rows of the batch that the backward walks at a time (no time split)."""
    ln = 2 if Ns <= 8 else 4 if Ns <= 16 else 8 if Ns <= 32 else 16 if Ns <= 64 else 32
    tiles = -(-D // ((256 if ln >= 16 else 128) // ln * 2))
    total = _lib.load().m3_selective_bwd_workspace_bytes(_lib.SelDesc(B, L, D, Ns, 0, 1))
    bc = -(-tiles * B * L * 8 * 4 * ln // 256) * 256
    return (total - bc) // (D * (4 * ln + 2) * 4)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,L,D,Ns,opt", [
    (1500, 33, 20, 8, dict(state=True)),
    (1201, 17, 33, 16, dict()),
    (1100, 20, 30, 24, dict(gate=False)),
    (500, 18, 40, 40, dict(state=True)),
    (400, 17, 20, 100, dict(skip=False, bias=False)),
])
def test_scan_over_many_rows(B, L, D, Ns, opt, dtype):
    """Ragged, with rows of length 0 between full ones."""
    assert B > 2 * _scan_bgroups(B, L, D, Ns) > 0
    a, gr = _scan_inputs(B, L, D, Ns, T[dtype], ragged=True, seed=B + Ns, **opt)
    a["lengths"][::3], a["lengths"][1::5] = L, 0
    _check_scan(a, gr, _run_scan(a, gr))


def test_scan_over_many_rows_split_along_time():
    """Long rows, split along time, and more of them than one turn holds."""
    a, gr = _scan_inputs(130, 1500, 20, 8, torch.float32, ragged=True, state=True, seed=7)
    a["lengths"][::3], a["lengths"][1::5] = 1500, 0
    _check_scan(a, gr, _run_scan(a, gr))
