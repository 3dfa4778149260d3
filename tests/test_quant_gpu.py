"""The product with 4-bit weights against its definition in 64 bits."""

import pytest
import torch

from redpanda_b200 import quant as Q
from seq_oracle import E, half_step
from test_quant import made

pytestmark = pytest.mark.gpu
T = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-5


def product(x, w, bias, norm_w, residual, silu_cols):
    """(out, bound) in 64 bits.  Every product is exact; a path to the sum passes
    the tensor core's additions of its group (8 instructions, at most 2^-22 of the
    largest term each: the unit cuts what lies below its 24 or more bits), the scale,
    three parts and at most groups / 8 + 8 + 3 additions of fp32, the norm's factor
    (sums of squares: K / 16 + 16 additions, halved by the root), bias and residual.
    The magnitudes are those of scale (q - 8) x and center x apart, bounded by
    (|w| + 16 scale) |x| through ``spread``."""
    xd, wd = x.double(), w["w"].double()
    k = xd.shape[1]
    n = k / 8 / w["group"] + 8 + 3 + 8
    rel = 0.0
    if norm_w is not None:
        xd = xd * (xd.square().mean(1, keepdim=True) + EPS) ** -0.5 * norm_w.double()
        rel = (k / 32 + 16 + 4) * E
    mag = xd.abs() @ w["spread"].double().T
    out = xd @ wd.T
    tol = (n * E + 8 * 4 * E + rel) * mag
    for t in (bias, residual):
        if t is not None:
            out = out + t.double()
            tol = tol + 2 * E * out.abs() + E * t.double().abs()
    if silu_cols:
        u = out[:, :silu_cols]
        s = torch.sigmoid(u)
        tol[:, :silu_cols] = tol[:, :silu_cols] * 1.1 + 4 * E * (u * s).abs() + 4 * E * u.abs() * s
        out = torch.cat([u * s, out[:, silu_cols:]], 1)
    return out, tol


def weight(n, k, group, center, seed):
    codes, scale, mid, w = made(n, k, group, center, seed)
    scale, mid = scale * 0.1, None if mid is None else mid * 0.1
    q = Q.Q4Weight.from_codes(codes, scale, mid, group)
    w = q.dequantize()
    wide = scale.float().repeat_interleave(group, 1)[:, :k]
    spread = (codes - 8).abs().float() * wide
    if mid is not None:
        spread = spread + mid.float().abs().repeat_interleave(group, 1)[:, :k]
    return q.to("cuda"), dict(w=w, spread=spread, group=group)


def run(rows, k, n, group, center, ty, norm=False, bias=True, res=False, split=None, silu=False,
        seed=0):
    ty = T[ty]
    g = torch.Generator().manual_seed(seed + rows + k + n)
    q, w = weight(n, k, group, center, seed + 1)
    x = torch.randn(rows, k, generator=g).to(ty)
    b = torch.randn(n, generator=g) if bias else None
    nw = torch.randn(k, generator=g) * 0.3 + 1 if norm else None
    r = torch.randn(rows, n, generator=g).to(ty) if res else None
    c = lambda t: None if t is None else t.cuda()  # noqa: E731
    got = Q.m3_rows_linear_q4(c(x), q, c(b), norm_weight=c(nw), eps=EPS, residual=c(r),
                              split=split, silu=silu)
    cut = n if split is None else split
    assert (got[0] is None) == (cut == 0) and (got[1] is None) == (cut == n)
    out = torch.cat([t for t in got if t is not None], 1)
    assert out.dtype == ty and out.shape == (rows, n)
    ref, tol = product(x, w, b, nw, r, cut if silu else 0)
    far = (out.cpu().double() - ref).abs()
    assert (far <= tol * 1.01 + half_step(ty) * (ref.abs() + tol)).all(), float((far / tol).max())


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("center", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,k,n", [(1, 1, 1), (1, 64, 16), (2, 384, 100), (3, 97, 33),
                                      (8, 768, 17), (5, 1000, 40), (1, 2311, 16)])
def test_matches_definition(rows, k, n, group, center, ty):
    run(rows, k, n, group, center, ty)


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("rows", range(1, 9))
def test_every_number_of_rows_with_all_around_it(rows, ty):
    run(rows, 200, 70, 64, True, ty, norm=True, res=True, split=30, silu=True, seed=rows)
    run(rows, 130, 50, 32, False, ty, norm=True, bias=False, seed=rows)


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("rows,k,n,group,center", [(8, 8192, 40, 32, True), (7, 5000, 64, 128, True),
                                                   (1, 65536, 20, 64, True),
                                                   (8, 65530, 18, 32, True),
                                                   (3, 256, 9600, 64, False),
                                                   (8, 320, 20001, 128, True),
                                                   (2, 64, 70000, 32, True)])
def test_large(rows, k, n, group, center, ty):
    """Inputs staged in parts, and tiles split over warps and CTAs."""
    run(rows, k, n, group, center, ty, norm=True)


@pytest.mark.parametrize("ty,k,rows", [("f32", 130, 3), ("bf16", 300, 5)])
@pytest.mark.parametrize("n", [11000, 27001, 34000, 45007, 50000, 64999, 75001, 80000])
def test_every_number_of_warps_along_the_outputs(n, ty, k, rows):
    """Tiles that fill one wave of CTAs with 2 to 8 warps' worth each, and more than one."""
    run(rows, k, n, 64, True, ty, norm=True, split=n // 3, silu=True)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("rows", [1, 4, 8])
@pytest.mark.parametrize("k,ld,off", [(130, 130, 0), (1002, 1002, 0), (1001, 1001, 0), (3, 3, 0),
                                      (2, 2, 0), (515, 520, 0), (515, 520, 1), (514, 518, 1),
                                      (514, 518, 2), (1000, 1009, 9), (7050, 7050, 0),
                                      (4985, 4987, 1)])
def test_bf16_rows_of_every_alignment(k, ld, off, rows, norm):
    """Rows that 16 bytes, words or elements may be copied from, that end inside them."""
    g = torch.Generator().manual_seed(k + rows)
    q, w = weight(40, k, 64, True, 3)
    base = torch.randn(rows * ld + off, generator=g).to(torch.bfloat16)
    cut = lambda t: t[off:].view(rows, ld)[:, :k]  # noqa: E731
    nw = torch.randn(k, generator=g) * 0.3 + 1 if norm else None
    got = Q.m3_rows_linear_q4(cut(base.cuda()), q, norm_weight=nw.cuda() if norm else None,
                              eps=EPS)[0]
    ref, tol = product(cut(base), w, None, nw, None, 0)
    far = (got.cpu().double() - ref).abs()
    assert (far <= tol * 1.01 + half_step(torch.bfloat16) * (ref.abs() + tol)).all()


def test_strides_split_ends_and_the_residual_in_place():
    g = torch.Generator().manual_seed(4)
    q, w = weight(48, 96, 32, True, 7)
    base = torch.randn(4, 300, generator=g)
    for off in (0, 1, 2, 5):                           # rows that pairs can and cannot be read from
        x = base[:, off:off + 96]
        ref, tol = product(x, w, None, None, None, 0)
        for split in (0, 48):
            got = Q.m3_rows_linear_q4(base.cuda()[:, off:off + 96], q, split=split)
            out = got[0] if split else got[1]
            assert ((out.cpu().double() - ref).abs() <= tol * 1.01).all()
    x, r = base[:, :96], base[:, 100:148]
    ref, tol = product(x, w, None, None, r, 0)
    stream = r.cuda()
    out, _ = Q.m3_rows_linear_q4(x.cuda(), q, residual=stream, out0=stream)
    assert out is stream
    assert ((stream.cpu().double() - ref).abs() <= tol * 1.01).all()
    wide = torch.full((4, 100), 3.0, device="cuda")    # outputs with a stride: nothing else moves
    Q.m3_rows_linear_q4(x.cuda(), q, residual=r.cuda(), out0=wide[:, :48])
    assert ((wide[:, :48].cpu().double() - ref).abs() <= tol * 1.01).all()
    assert (wide[:, 48:] == 3).all()


def test_overlaps_are_refused():
    q, _ = weight(48, 48, 32, True, 7)
    x = torch.zeros(3, 48, device="cuda")
    with pytest.raises(RuntimeError):
        Q.m3_rows_linear_q4(x, q, out0=x)
    buf = torch.zeros(4, 48, device="cuda")
    with pytest.raises(RuntimeError):
        Q.m3_rows_linear_q4(x, q, residual=buf[:3], out0=buf[1:])
    with pytest.raises(ValueError):
        Q.m3_rows_linear_q4(x, q, out0=torch.zeros(3, 47, device="cuda"))
    with pytest.raises(ValueError):
        Q.m3_rows_linear_q4(x, q, residual=torch.zeros(3, 48, device="cuda").bfloat16())


def test_no_rows_infinities_and_nan():
    q, w = weight(40, 70, 32, False, 3)
    assert Q.m3_rows_linear_q4(torch.zeros(0, 70, device="cuda"), q)[0].shape == (0, 40)
    x = torch.randn(4, 70, generator=torch.Generator().manual_seed(1))
    x[1, 5], x[2, 9] = float("inf"), float("nan")
    x[3] = 3e38
    out = Q.m3_rows_linear_q4(x.cuda(), q)[0].cpu()
    ref = x[0].double() @ w["w"].double().T
    assert ((out[0].double() - ref).abs() <= 60 * E * (x[0].abs().double() @ w["spread"].double().T)
            ).all()                                    # one row's values are no other's
    live = w["w"][:, 5] != 0
    assert torch.equal(out[1][live], torch.sign(w["w"][live, 5]) * float("inf"))
    assert torch.isnan(out[2]).all()


def test_another_stream_and_capture():
    q, _ = weight(300, 256, 64, True, 11)
    x = torch.randn(4, 256, generator=torch.Generator().manual_seed(2)).cuda()

    def once():
        a, _ = Q.m3_rows_linear_q4(x, q, silu=True, overlap=True)
        return Q.m3_rows_linear_q4(a[:, :256], q, overlap=True)[0]
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
    assert torch.equal(first, second) and torch.equal(first, third)


def test_one_weight_on_two_streams_and_replays_of_changed_rows():
    q, _ = weight(700, 600, 64, True, 15)
    xs = torch.randn(6, 3, 600, generator=torch.Generator().manual_seed(5)).cuda()
    alone = [Q.m3_rows_linear_q4(x, q)[0] for x in xs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = {}
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for i, x in enumerate(xs):
        with torch.cuda.stream(streams[i % 2]):
            got[i] = Q.m3_rows_linear_q4(x, q, overlap=True)[0]
    torch.cuda.synchronize()
    assert all(torch.equal(got[i], alone[i]) for i in got)
    static, graph = xs[0].clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = Q.m3_rows_linear_q4(static, q)[0]
    for x, ref in zip(xs, alone):
        static.copy_(x)
        graph.replay()
        assert torch.equal(out, ref)


@pytest.mark.parametrize("ty", ["f32", "bf16"])
def test_quantized_weight_and_its_product(ty):
    """From a float weight to a product: what the dequantised weight gives."""
    g = torch.Generator().manual_seed(1)
    w, x = torch.randn(300, 200, generator=g), torch.randn(5, 200, generator=g).to(T[ty])
    q = Q.Q4Weight.quantize(w, 32)
    d = q.dequantize()
    scale = (d.abs().amax(1, keepdim=True) * 2).expand_as(d)     # >= |q - 8| scale + |center|
    out = Q.m3_rows_linear_q4(x.cuda(), q.to("cuda"))[0]
    ref, tol = product(x, dict(w=d, spread=scale, group=32), None, None, None, 0)
    far = (out.cpu().double() - ref).abs()
    assert (far <= tol * 1.01 + half_step(T[ty]) * (ref.abs() + tol)).all()


def norm_in_chunks(rows, k, n, group, center, ty):
    """The product with the norm ahead, on the GPU; every 13th output against the
    definition (13 and a tile's 16 have no common divisor), whose columns all count in
    the row's mean square."""
    g = torch.Generator("cuda").manual_seed(rows + k + n + group)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    codes = torch.randint(0, 16, (n, k), generator=g, device="cuda", dtype=torch.uint8)
    scale = torch.rand(n, -(-k // group), generator=g, device="cuda").add_(0.1).mul_(0.1).bfloat16()
    mid = rnd(*scale.shape).mul_(0.1).bfloat16() if center else None
    x, b, nw = rnd(rows, k).to(T[ty]), rnd(n), rnd(k) * 0.3 + 1
    q = Q.Q4Weight.from_codes(codes, scale, mid, group)
    out = Q.m3_rows_linear_q4(x, q, b, norm_weight=nw, eps=EPS)[0]
    at = torch.arange(0, n, 13, device="cuda")
    wide = lambda t: t[at].double().repeat_interleave(group, 1)[:, :k]  # noqa: E731
    w = (codes[at].double() - 8) * wide(scale)
    spread = w.abs()
    if center:
        w, spread = w + wide(mid), spread + wide(mid).abs()
    ref, tol = product(x, dict(w=w, spread=spread, group=group), b[at], nw, None, 0)
    far = (out[:, at].double() - ref).abs()
    assert (far <= tol * 1.01 + half_step(T[ty]) * (ref.abs() + tol)).all(), float((far / tol).max())


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("rows,k,n,group", [(8, 2048, 50304, 64), (2, 8192, 40000, 64),
                                            (8, 3000, 65536, 32), (8, 8192, 40000, 32),
                                            (4, 4096, 50304, 32)])
def test_norm_over_inputs_staged_in_parts(rows, k, n, group, ty):
    """One warp along the columns, and inputs that are staged in two to six parts."""
    norm_in_chunks(rows, k, n, group, True, ty)


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n", [9000, 16000, 27001, 34000, 45007, 50000, 64999, 75001])
def test_norm_for_every_number_of_warps_and_parts(n, group, ty):
    """1 to 8 warps' worth of tiles; inputs in one part and in two to five."""
    for rows, k in ((8, 2048), (8, 3001), (5, 4100), (8, 4992)):
        norm_in_chunks(rows, k, n, group, (n + k) % 2 == 0, ty)


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("norm", [False, True])
def test_rows_that_are_not_finite_change_no_other(norm, ty):
    """With centers an infinity's outputs are infinite or NaN; the other rows keep their
    bits."""
    q, w = weight(200, 300, 64, True, 5)
    g = torch.Generator().manual_seed(8)
    x = torch.randn(6, 300, generator=g).to(T[ty]).cuda()
    nw = torch.randn(300, generator=g).cuda() if norm else None
    good = Q.m3_rows_linear_q4(x, q, norm_weight=nw, eps=EPS)[0]
    x[1, 17], x[4, 299], x[2, 64] = float("inf"), float("-inf"), float("nan")
    out = Q.m3_rows_linear_q4(x, q, norm_weight=nw, eps=EPS)[0]
    keep = [0, 3, 5]
    assert torch.equal(out[keep], good[keep])
    for row, col in ((1, 17), (4, 299), (2, 64)):
        assert not torch.isfinite(out[row][w["w"][:, col].cuda() != 0]).any()
