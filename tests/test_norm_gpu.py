"""Layer and RMS norm kernels against their definition in 64 bits."""

import pytest
import torch

import seq_oracle as O
from redpanda_b200 import norm as N

pytestmark = pytest.mark.gpu
T = {"f32": torch.float32, "bf16": torch.bfloat16}


def _inputs(rows, d, tx, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, d, generator=g) * spread + 0.5).to(tx)
    w = torch.randn(d, generator=g) * 0.3 + 1
    b = torch.randn(d, generator=g) * 0.3
    return x, w, b, torch.randn(rows, d, generator=g)


def _check(x, w, b, gr, eps, rms, ty, y, dx=None, dw=None, db=None):
    """k e bounds: statistics are sums of d terms in trees of depth < 32 + 32
    (32 per thread, then shuffles and warps) on squares and differences; rsqrt 2
    ulp; then a handful of products: k = 96 covers every path."""
    k, e = 96, O.E
    ref = O.norm(x, w, b, eps, rms, gr)
    ry, rdx, rdw, rdb = ref
    xd = x.double()
    mu = 0 if rms else xd.mean(1, keepdim=True)
    mag = xd.abs() + (0 if rms else xd.abs().mean(1, keepdim=True))
    r = ((xd - mu).square().mean(1, keepdim=True) + eps) ** -0.5
    # |x - mu| is off by a rounding of x and mu; xh by that and r's error
    mxh = mag * r
    my = mxh * w.double().abs() + (0 if b is None else b.double().abs())
    tol = k * e * my + O.half_step(ty) * ry.abs()
    assert ((y.cpu().double() - ry).abs() <= tol).all()
    if dx is None:
        return
    g = gr.double()
    q = (g * w.double()).abs()
    amp = (mag * r).square().mean(1, keepdim=True).clamp(min=1.0)   # error of r through xh
    mdx = r * (q + q.mean(1, keepdim=True) + mxh * (q * mxh).mean(1, keepdim=True)) * amp
    assert ((dx.cpu().double() - rdx).abs()
            <= k * e * mdx + O.half_step(x.dtype) * rdx.abs()).all()
    # sums over the rows: one addition per row at most, beside the row's own error
    rows = x.shape[0]
    assert ((dw.cpu().double() - rdw).abs() <= (k + rows) * e * (g.abs() * mxh).sum(0)).all()
    if db is not None:
        assert ((db.cpu().double() - rdb).abs() <= (8 + rows) * e * g.abs().sum(0)).all()


@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("tx,ty", [("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16"),
                                   ("bf16", "f32")])
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 2), (5, 31), (700, 64), (9, 257), (33, 1000),
                                    (17, 1024), (5, 1028), (6, 1030), (3, 4096), (3, 4100),
                                    (2, 16384), (2, 16388), (1, 32767)])
def test_norm_matches_definition(rows, d, tx, ty, rms):
    tx, ty = T[tx], T[ty]
    x, w, b, g = _inputs(rows, d, tx, rows * 7 + d)
    g = g.to(ty)
    xc, wc, bc = (t.cuda().requires_grad_(True) for t in (x, w, b))
    if rms:
        b = None
        y = N.m3_rms_norm(xc, wc, eps=1e-5, out_dtype=ty)
        dx, dw = torch.autograd.grad(y, (xc, wc), g.cuda())
        db = None
    else:
        y = N.m3_layer_norm(xc, wc, bc, eps=1e-5, out_dtype=ty)
        dx, dw, db = torch.autograd.grad(y, (xc, wc, bc), g.cuda())
    assert y.dtype == ty and dx.dtype == tx
    _check(x, w, b, g, 1e-5, rms, ty, y.detach(), dx, dw, db)
    with torch.no_grad():   # the inference call gives the same bits
        y2 = (N.m3_rms_norm(xc, wc, eps=1e-5, out_dtype=ty) if rms
              else N.m3_layer_norm(xc, wc, bc, eps=1e-5, out_dtype=ty))
    assert torch.equal(y, y2)


def test_norm_strides_and_leading_dimensions():
    g = torch.Generator().manual_seed(0)
    base = torch.randn(4, 6, 200, generator=g)
    w, b = torch.randn(72, generator=g), torch.randn(72, generator=g)
    for off in (0, 3, 64):   # 3: rows that no vector load can start at (another order of sums)
        view = base[..., off:off + 72]
        y = N.m3_layer_norm(base.cuda()[..., off:off + 72], w.cuda(), b.cuda())
        assert y.shape == (4, 6, 72)
        _check(view.reshape(24, 72), w, b, torch.zeros(24, 72), 1e-5, False, torch.float32,
               y.reshape(24, 72))
        if off != 3:
            assert torch.equal(y, N.m3_layer_norm(view.contiguous().cuda(), w.cuda(), b.cuda()))
    # an expanded row, and a tensor whose last dimension is not contiguous
    one = base[0, :1, :72].cuda()
    y = N.m3_rms_norm(one.expand(5, 72), w.cuda())
    assert torch.equal(y, N.m3_rms_norm(one, w.cuda()).expand(5, 72))
    tr = base[0].cuda().t()[:72]                       # (72, 6)
    w6 = torch.ones(6, device="cuda")
    assert torch.equal(N.m3_rms_norm(tr, w6), N.m3_rms_norm(tr.contiguous(), w6))


def test_norm_gradient_of_a_broadcast_row():
    """The gradient of an expanded input is the sum over its copies."""
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(1, 40, generator=g), torch.randn(40, generator=g)
    up = torch.randn(7, 40, generator=g)
    xc = x.cuda().requires_grad_(True)
    (dx,) = torch.autograd.grad(N.m3_rms_norm(xc.expand(7, 40), w.cuda()), xc, up.cuda())
    ref = O.norm(x.expand(7, 40), w, None, 1e-5, True, up)[1].sum(0, keepdim=True)
    r = x.double().square().mean().add(1e-5).rsqrt()
    mag = 4 * r * (up.abs().sum(0) * w.abs()).max().double() * 40 ** 0.5
    assert ((dx.cpu().double() - ref).abs() <= 110 * O.E * mag).all()


def test_norm_large_mean_keeps_the_variance():
    """Rows at 1000 with a spread of 1: mean(x^2) - mean^2 would lose 20 bits."""
    x, w, b, _ = _inputs(16, 512, torch.float32, 3)
    x = x + 1000
    y = N.m3_layer_norm(x.cuda(), w.cuda(), b.cuda()).cpu().double()
    ry = O.norm(x, w, b, 1e-5, False)
    # x - mean is off by a rounding of the mean's sums: 40 e * 1000, here 2.4e-3
    assert (y - ry).abs().max() <= 40 * O.E * 1000 * w.abs().max() * 1.2


def test_norm_gradient_against_differences():
    x, w, b, g = _inputs(6, 48, torch.float32, 5)
    xc, wc, bc = (t.cuda().requires_grad_(True) for t in (x, w, b))
    grads = torch.autograd.grad(N.m3_layer_norm(xc, wc, bc), (xc, wc, bc), g.cuda())
    gen = torch.Generator().manual_seed(6)
    for i, t in enumerate((x, w, b)):
        v = torch.randn(t.shape, generator=gen).double()
        h, args = 1e-4, [x.double(), w.double(), b.double()]
        f = []
        for sgn in (1, -1):
            a = list(args)
            a[i] = a[i] + sgn * h * v
            f.append((O.norm(a[0], a[1], a[2], 1e-5, False) * g.double()).sum())
        diff = ((f[0] - f[1]) / (2 * h)).item()
        ours = (grads[i].cpu().double() * v).sum().item()
        scale = (grads[i].cpu().double() * v).abs().sum().item()
        assert abs(ours - diff) <= 1e-5 * scale      # h^2 of a smooth function, and 96 e


def test_norm_empty_and_refusals():
    w = torch.ones(8, device="cuda", requires_grad=True)
    x = torch.zeros(0, 8, device="cuda", requires_grad=True)
    y = N.m3_layer_norm(x, w)
    assert y.shape == (0, 8)
    dx, dw = torch.autograd.grad(y.sum(), (x, w))
    assert dx.shape == (0, 8) and not dw.any()
    with pytest.raises(RuntimeError, match="one device|CUDA"):
        N.m3_rms_norm(torch.zeros(2, 8), w)
    with pytest.raises(TypeError):
        N.m3_rms_norm(torch.zeros(2, 8, device="cuda", dtype=torch.float16), w)


def test_norm_is_deterministic_and_capturable():
    x, w, b, g = (t.cuda() for t in _inputs(5000, 96, torch.float32, 9))

    def once():
        xc, wc, bc = (t.detach().requires_grad_(True) for t in (x, w, b))
        y = N.m3_layer_norm(xc, wc, bc)
        return (y.detach(), *torch.autograd.grad(y, (xc, wc, bc), g))
    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):      # another stream, then a capture
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = once()
    graph.replay()
    for a, c, d in zip(first, second, third):
        assert torch.equal(a, c) and torch.equal(a, d)


def test_layer_norm_module():
    m = N.LayerNorm(64).cuda()
    x = torch.randn(10, 64, device="cuda")
    ref = torch.nn.functional.layer_norm(x, (64,), m.weight, m.bias, m.eps)
    assert torch.equal(m(x), ref)                      # off: torch's own
    m.use_kernel = True
    assert torch.equal(m(x), N.m3_layer_norm(x, m.weight, m.bias, m.eps))
    assert set(m.state_dict()) == {"weight", "bias"}


def test_layer_norm_module_under_autocast():
    """float32 results under autocast, as torch's layer norm, for bfloat16 inputs."""
    m = N.LayerNorm(64).cuda()
    x = torch.randn(10, 64, generator=torch.Generator().manual_seed(8)).cuda().bfloat16()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        ref = m(x)
        m.use_kernel = True
        got = m(x)
    assert got.dtype == ref.dtype == torch.float32
    # sums of 64 terms in either order and a dozen roundings: each side is off by
    # at most (64 + 12) 2^-24 of |y| + max |x - mean| rstd < 8, twice
    assert (got - ref).abs().max().item() <= 2 * 76 * 2 ** -24 * 16
