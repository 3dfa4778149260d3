"""The gated linear recurrence against its definition in 64 bits."""

import math

import pytest
import torch

import layer_oracle as O
from redpanda_b200 import gated as G

pytestmark = pytest.mark.gpu
T = {"f32": torch.float32, "bf16": torch.bfloat16}


def inputs(B, L, D, ty, seed, state=False, ragged=False, spread=2.0):
    g = torch.Generator().manual_seed(seed)

    def n(*s, k=1.0):
        return torch.randn(*s, generator=g) * k

    x, g1, g2, gr = (n(B, L, D, k=k).to(ty) for k in (1.0, spread, spread, 1.0))
    decay = n(D, k=1.5) - 3
    st = n(B, D) if state else None
    lens = None
    if ragged:
        lens = torch.randint(0, L + 1, (B,), generator=g)
        lens[0] = L
        lens[-1] = 0 if B > 1 else L
    return x, g1, g2, decay, gr, st, lens


def cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


def check(x, rg, ig, decay, gr, st, lens, c=8.0):
    ty = x.dtype
    ref = O.gated(x, rg, ig, decay, c, st, lens, gr)
    dx, dr, di, dd, dg, ds, dl = cuda(x, rg, ig, decay, gr, st, lens)
    y0, h = G.m3_gated_scan_with_state(dx, dr, di, dd, c=c, state=ds, lengths=dl)
    leaves = [t.requires_grad_(True) for t in (dx, dr, di, dd)]
    y = G.m3_gated_scan(*leaves, c=c, state=ds, lengths=dl)
    grads = torch.autograd.grad(y, leaves, dg)
    assert torch.equal(y, y0)
    far = {"y": O.excess(y, ref["y"], ref["+y"], ty), "h": O.excess(h, ref["h"], ref["+h"],
                                                                    torch.float32)}
    for k, t in zip(("dx", "drg", "dig", "ddecay"), grads):
        assert t.dtype == (torch.float32 if k == "ddecay" else ty)
        far[k] = O.excess(t, ref[k], ref["+" + k], t.dtype)
    assert max(far.values()) <= 1, far


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("B,L,D", [(1, 1, 1), (2, 1, 64), (3, 7, 65), (1, 8, 2), (2, 9, 128),
                                   (5, 64, 96), (3, 65, 72), (2, 130, 200), (1, 1025, 64),
                                   (1, 2050, 8), (2, 777, 33), (300, 5, 64)])
def test_matches_definition(B, L, D, ty):
    check(*inputs(B, L, D, T[ty], 3 * B + L + D))


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("B,L,D", [(4, 33, 64), (7, 150, 40), (3, 1300, 64), (2, 1, 16)])
def test_states_and_lengths(B, L, D, ty):
    check(*inputs(B, L, D, T[ty], B + L + D, state=True, ragged=True))


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("B,D", [(1, 1), (3, 64), (17, 33), (400, 132)])
def test_step_matches_definition(B, D, ty):
    x, rg, ig, decay, _, st, _ = inputs(B, 1, D, T[ty], B + D, state=True)
    ref = O.gated(x, rg, ig, decay, 8.0, st)
    h, gates = st.cuda(), torch.cat([rg, ig], 2)[:, 0].cuda()
    with torch.no_grad():
        y = G.m3_gated_step_(h, x[:, 0].cuda(), gates[:, :D], gates[:, D:], decay.cuda())
    assert O.excess(h, ref["h"], ref["+h"], torch.float32) <= 1
    assert y.dtype == T[ty] and O.excess(y, ref["y"][:, 0], ref["+y"][:, 0], T[ty]) <= 1


def test_steps_continue_a_prompt_and_parts_continue_each_other():
    """A sequence in one call, in two with the state between, and token by token."""
    x, rg, ig, decay, _, _, _ = cuda(*inputs(2, 90, 48, torch.float32, 5))
    ref = O.gated(*(t.cpu() for t in (x, rg, ig, decay)))
    with torch.no_grad():
        y1, h = G.m3_gated_scan_with_state(x[:, :37], rg[:, :37], ig[:, :37], decay)
        y2, h2 = G.m3_gated_scan_with_state(x[:, 37:60], rg[:, 37:60], ig[:, 37:60], decay, state=h)
        ys = [G.m3_gated_step_(h2, x[:, t], rg[:, t], ig[:, t], decay) for t in range(60, 90)]
    y = torch.cat([y1, y2, torch.stack(ys, 1)], 1)
    assert O.excess(y, ref["y"], ref["+y"], torch.float32) <= 1
    assert O.excess(h2, ref["h"], ref["+h"], torch.float32) <= 1


@pytest.mark.parametrize("ty", ["f32", "bf16"])
def test_strided_views_mixed_types_and_broadcast_gradient(ty):
    ty = T[ty]
    g = torch.Generator().manual_seed(2)
    base = torch.randn(3, 41, 200, generator=g).to(ty)
    decay, up = torch.randn(48, generator=g) - 3, torch.randn(3, 41, 48, generator=g).to(ty)
    for off in ((0, 64, 128), (1, 50, 100)):           # 16-byte rows, and rows that are not
        views = [base[..., o:o + 48] for o in off]
        ref = O.gated(*views, decay, g=up)
        b = base.cuda().requires_grad_(True)
        dd = decay.cuda().requires_grad_(True)
        y = G.m3_gated_scan(*(b[..., o:o + 48] for o in off), dd)
        assert O.excess(y, ref["y"], ref["+y"], ty) <= 1
        db, ddec = torch.autograd.grad(y, (b, dd), up.cuda())
        for o, k in zip(off, ("dx", "drg", "dig")):
            assert O.excess(db[..., o:o + 48], ref[k], ref["+" + k], ty) <= 1
        assert O.excess(ddec, ref["ddecay"], ref["+ddecay"], torch.float32) <= 1
    # one gate row for the whole batch: its gradient is the sum over the rows
    x, rg, ig = (base[..., o:o + 48].float() for o in (0, 64, 128))
    one = rg[:1].cuda().requires_grad_(True)
    (dr,) = torch.autograd.grad(G.m3_gated_scan(x.cuda(), one.expand(3, 41, 48), ig.cuda(),
                                                decay.cuda()), one, up.float().cuda())
    ref = O.gated(x, rg[:1].expand(3, 41, 48), ig, decay, g=up.float())
    tot = ref["drg"].sum(0, keepdim=True)
    assert O.excess(dr, tot, ref["+drg"].sum(0, keepdim=True)
                    + 4 * O.E * ref["drg"].abs().sum(0, keepdim=True), torch.float32) <= 1
    # types that differ: float32 for all
    y = G.m3_gated_scan(x.cuda().bfloat16(), rg.cuda(), ig.cuda().bfloat16(), decay.cuda())
    assert y.dtype == torch.float32


def test_extreme_gates():
    """Gates shut and open as far as the type goes, decays of 0 and of everything:
    finite results where the definition has them."""
    v = torch.tensor([-1e4, -100.0, -90.0, -40.0, -20.0, -5.0, 0.0, 5.0, 20.0, 90.0, 1e4])
    rg, ig = v.repeat_interleave(11).view(1, 121, 1), v.repeat(11).view(1, 121, 1)
    decay = torch.tensor([-200.0, -100.0, -30.0, -16.0, -14.0, -3.0, 0.0, 3.0, 30.0, 1e4])
    D = len(decay)
    x = torch.randn(1, 121, D, generator=torch.Generator().manual_seed(1))
    up = torch.randn(1, 121, D, generator=torch.Generator().manual_seed(2))
    rg, ig = rg.expand(1, 121, D).contiguous(), ig.expand(1, 121, D).contiguous()
    leaves = [t.cuda().requires_grad_(True) for t in (x, rg, ig, decay)]
    y = G.m3_gated_scan(*leaves)
    grads = torch.autograd.grad(y, leaves, up.cuda())
    ref = O.gated(x, rg, ig, decay, g=up)
    assert all(torch.isfinite(t).all() for t in (y, *grads))
    # A sigmoid below 2^-126 = 1.2e-38 is 0 in fp32 without subnormals.  With
    # c softplus(decay) = 8e4 that loses l up to 9.4e-34, so m = sqrt(2 l) up to
    # 4.4e-17: of an input of size |x|, and of what multiplies it in the gradients (q,
    # at most the sum of |up|; e, at most m / 2 times u x q).
    lost = 4.4e-17
    X, U = (t.double().abs().sum(1, keepdim=True) for t in (x, up))
    assert ((y.cpu().double() - ref["y"]).abs() <= 1.01 * ref["+y"] + lost * X).all()
    for k, t, size in zip(("dx", "drg", "dig"), grads, (U, U * X, U * X)):
        assert ((t.cpu().double() - ref[k]).abs() <= 1.01 * ref["+" + k] + lost * size).all(), k
    assert ((grads[3].cpu().double() - ref["ddecay"]).abs()
            <= 1.01 * ref["+ddecay"] + lost * 121 * (U * X)[0, 0]).all()


def test_long_memory_keeps_its_precision():
    """A decay of 0.9997 over 6000 steps: a one-signed error of the decay of 2e-8
    would be 7.5e-5 of the state.

    The bar: the gate is the same at every step, so the rounding of a itself, up to
    2^-25, is one-signed here and shifts the state by that over 1 - a = 2.66e-4; the
    shift is what rounding this a to fp32 gives.  Beside it, the roundings of the
    state and of the runs' products (two per step, independent, 2^-25 / sqrt(3) of the
    state each) over 1 / (2 (1 - a)) = 1880 steps: sqrt(2 * 1880) * 1.7e-8 = 1.1e-6;
    four times that."""
    g = torch.Generator().manual_seed(3)
    x = torch.rand(1, 6000, 4, generator=g)
    rg, ig = torch.full_like(x, 1.0), torch.zeros_like(x)
    decay = torch.full((4,), -10.0)
    y, h = G.m3_gated_scan_with_state(*cuda(x, rg, ig, decay))
    ref = O.gated(x, rg, ig, decay)
    a = math.exp(-8 * math.log1p(math.exp(-10)) / (1 + math.exp(-1)))
    shift = abs(float(torch.tensor(a, dtype=torch.float32)) - a) / (1 - a)
    assert ((h.cpu().double() - ref["h"]).abs() / ref["h"].abs()).max() < shift + 4.4e-6
    assert O.excess(y, ref["y"], ref["+y"], torch.float32) <= 1


def test_steps_past_a_length_are_not_read():
    x, rg, ig, decay, gr, st, lens = inputs(4, 30, 40, torch.float32, 8, True, True)
    bad = [t.clone() for t in (x, rg, ig, gr)]
    for i, n in enumerate(lens.tolist()):
        for t, v in zip(bad, (float("nan"), float("inf"), float("-inf"), float("nan"))):
            t[i, n:] = v
    res = []
    for a, b, c, up in ((x, rg, ig, gr), bad):
        leaves = [t.cuda().requires_grad_(True) for t in (a, b, c, decay)]
        y = G.m3_gated_scan(*leaves, state=st.cuda(), lengths=lens.cuda())
        _, h = G.m3_gated_scan_with_state(*(t.detach() for t in leaves), state=st.cuda(),
                                          lengths=lens.cuda())
        res.append([y.detach(), h, *torch.autograd.grad(y, leaves, up.cuda())])
    for a, b in zip(*res):
        assert torch.equal(a, b)
    for i, n in enumerate(lens.tolist()):
        assert not res[0][0][i, n:].any()
    # lengths past L and below 0 count as L and 0
    odd = torch.tensor([99, -3, 30, 0])
    y = G.m3_gated_scan(*cuda(x, rg, ig, decay), lengths=odd.cuda())
    assert torch.equal(y, G.m3_gated_scan(*cuda(x, rg, ig, decay),
                                          lengths=odd.clamp(0, 30).cuda()))


def test_nan_stays_in_its_channel():
    x, rg, ig, decay, _, _, _ = inputs(1, 20, 6, torch.float32, 4)
    rg[0, 7, 2], x[0, 3, 5], ig[0, 11, 0] = (float("nan"),) * 3
    y = G.m3_gated_scan(*cuda(x, rg, ig, decay)).cpu()[0]
    for c, t in ((2, 7), (5, 3), (0, 11)):
        assert not torch.isnan(y[:t, c]).any() and torch.isnan(y[t:, c]).all()
    assert not torch.isnan(y[:, [1, 3, 4]]).any()


def test_gradient_against_differences():
    x, rg, ig, decay, gr, st, _ = inputs(2, 13, 5, torch.float32, 6, state=True, spread=1.0)
    leaves = [t.cuda().requires_grad_(True) for t in (x, rg, ig, decay)]
    grads = torch.autograd.grad(G.m3_gated_scan(*leaves, state=st.cuda()), leaves, gr.cuda())
    gen = torch.Generator().manual_seed(7)
    args = [t.double() for t in (x, rg, ig, decay)]
    for i in range(4):
        v, h, f = torch.randn(args[i].shape, generator=gen).double(), 1e-5, []
        for sign in (1, -1):
            moved = list(args)
            moved[i] = moved[i] + sign * h * v
            f.append((O.gated(*moved, state=st)["y"] * gr.double()).sum())
        diff = ((f[0] - f[1]) / (2 * h)).item()
        ours = grads[i].cpu().double() * v
        # h^2 times third derivatives (below 1e3), rounding / h = 1e-9, and the
        # gradients' own bound, 100 e of their paths
        assert abs(ours.sum().item() - diff) <= 1e-5 * ours.abs().sum().item() + 1e-7


def test_empty_batches_and_sequences():
    d = torch.zeros(8, device="cuda", requires_grad=True)
    for B, L in ((0, 5), (3, 0)):
        x = torch.zeros(B, L, 8, device="cuda", requires_grad=True)
        st = torch.ones(B, 8, device="cuda")
        y, h = G.m3_gated_scan_with_state(x, x, x, d, state=st)
        assert y.shape == (B, L, 8) and torch.equal(h, st)
        dx, dd = torch.autograd.grad(y.sum(), (x, d))
        assert dx.shape == x.shape and not dd.any()
    with torch.no_grad():
        assert G.m3_gated_step_(torch.zeros(0, 8, device="cuda"),
                                *3 * [torch.zeros(0, 8, device="cuda")], d).shape == (0, 8)


def test_another_stream_capture_and_side_by_side():
    a, b = (cuda(*inputs(3, 700, 64, torch.float32, s))[:5] for s in (1, 2))

    def once(x, rg, ig, decay, gr):
        leaves = [t.detach().requires_grad_(True) for t in (x, rg, ig, decay)]
        y = G.m3_gated_scan(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, gr)]
    first, other = once(*a), once(*b)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (s1, s2):
        s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s1):
        r1 = once(*a)
    with torch.cuda.stream(s2):
        r2 = once(*b)
    for s in (s1, s2):
        torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r3 = once(*a)
    graph.replay()
    for x, y, w in zip(first, r1, r3):
        assert torch.equal(x, y) and torch.equal(x, w)
    for x, y in zip(other, r2):
        assert torch.equal(x, y)


def test_state_version_moves_and_saved_states_raise():
    h = torch.zeros(2, 8, device="cuda")
    v = h._version
    with torch.no_grad():
        G.m3_gated_step_(h, *3 * [torch.ones(2, 8, device="cuda")], torch.zeros(8, device="cuda"))
    assert h._version > v


@pytest.mark.parametrize("ty", ["f32", "bf16"])
def test_many_rows_walked_by_one_cta(ty):
    """More rows than one wave of CTAs: each walks several, of other lengths."""
    check(*inputs(1500, 11, 64, T[ty], 4, state=True, ragged=True))


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 66, 67, 1])
def test_more_rows_than_warps(D, ty):
    """Rows and channel tiles for a warp each, forward (3552 and more)."""
    check(*inputs(3600, 9, D, T[ty], D, state=True, ragged=True))


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("B,L,D", [(1, 900, 1001), (2, 515, 130), (1, 4100, 63), (3, 40, 999)])
@pytest.mark.parametrize("offset", [0, 1, 2, 3])
def test_rows_of_every_alignment(B, L, D, offset, ty):
    """Views that start at every offset from 16 bytes, with strides of their own, and
    whose first and last elements are the storage's."""
    ty = T[ty]
    g = torch.Generator().manual_seed(D + offset)
    decay, up = torch.randn(D, generator=g) - 3, torch.randn(B, L, D, generator=g).to(ty)
    flat = [torch.randn(offset + B * L * (D + k) - k, generator=g).to(ty) for k in range(3)]

    def views(ts):
        return [t.as_strided((B, L, D), (L * (D + k), D + k, 1), offset) for k, t in enumerate(ts)]
    ref = O.gated(*views(flat), decay, g=up)
    base = [t.cuda().requires_grad_(True) for t in flat]
    dd = decay.cuda().requires_grad_(True)
    y = G.m3_gated_scan(*views(base), dd)
    assert O.excess(y, ref["y"], ref["+y"], ty) <= 1
    grads = torch.autograd.grad(y, (*base, dd), up.cuda())
    for t, k in zip(views(grads[:3]), ("dx", "drg", "dig")):
        assert O.excess(t, ref[k], ref["+" + k], ty) <= 1
    assert O.excess(grads[3], ref["ddecay"], ref["+ddecay"], torch.float32) <= 1


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("B,L,D", [(1, 1, 1), (3, 64, 96), (2, 777, 33), (1, 3000, 64),
                                   (2, 130, 200), (3600, 9, 64)])
def test_decays_near_one(B, L, D, ty):
    """Decays whose exponent needs no range reduction, in every channel of a warp."""
    x, rg, ig, _, gr, st, lens = inputs(B, L, D, T[ty], B + 3 * L + D, True, True)
    decay = torch.rand(D, generator=torch.Generator().manual_seed(D)) * 3 - 7
    check(x, rg, ig, decay, gr, st, lens)


@pytest.mark.parametrize("c", [0.5, 300.0])
def test_other_factors_of_the_decay(c):
    x, rg, ig, decay, gr, st, lens = inputs(2, 300, 70, torch.float32, 12, True, True)
    check(x, rg, ig, decay, gr, st, lens, c=c)


def test_rows_without_steps_among_long_ones():
    """Few long rows, split over clusters, of length 0 first, last, alone and all."""
    x, rg, ig, decay, gr, st, _ = inputs(4, 2500, 64, torch.float32, 13, True)
    for lens in ([0, 2500, 3, 0], [0, 0, 0, 0], [2500, 0, 0, 1], [0, 0, 0, 2500]):
        check(x, rg, ig, decay, gr, st, torch.tensor(lens))


def test_long_rows_side_by_side_on_two_streams():
    """Two calls whose clusters run at the same time give what each gives alone."""
    sets = [cuda(*inputs(1, 20000, 512, torch.bfloat16, s))[:5] for s in (21, 22)]

    def once(x, rg, ig, decay, gr):
        leaves = [t.detach().requires_grad_(True) for t in (x, rg, ig, decay)]
        y = G.m3_gated_scan(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, gr)]
    alone = [once(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(once(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for res in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(alone[i], res))


def test_replays_read_the_buffers_as_they_are_then():
    """A captured scan, its backward pass and a step replayed on changed inputs."""
    first, second = (cuda(*inputs(2, 900, 48, torch.float32, s, state=True))[:6] for s in (1, 2))
    static = [t.clone().requires_grad_(i < 4) for i, t in enumerate(first)]
    h = torch.zeros(2, 48, device="cuda")

    def run(x, rg, ig, decay, gr, st, h):
        y, last = G.m3_gated_scan_with_state(x, rg, ig, decay, state=st)
        grads = torch.autograd.grad(y, (x, rg, ig, decay), gr)
        with torch.no_grad():
            out = G.m3_gated_step_(h, x[:, 0], rg[:, 0], ig[:, 0], decay)
        return [y.detach(), last, *grads, out]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(*static, h)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(*static, h)
    for src in (second, first):
        with torch.no_grad():
            for a, b in zip(static, src):
                a.copy_(b)
        h.zero_()
        graph.replay()
        leaves = [t.clone().requires_grad_(i < 4) for i, t in enumerate(src)]
        for a, b in zip(out, run(*leaves, torch.zeros_like(h))):
            assert torch.equal(a, b)


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("D", [70, 72, 65, 127])
@pytest.mark.parametrize("far", [False, True])
def test_channels_do_not_depend_on_their_neighbours(D, far, ty):
    """A tile's last channels alone, or beside channels whose decays are near one or far
    from it: the same bits, whichever form of the decay the warp takes (rows enough for a
    warp each, so that nothing is joined)."""
    x, rg, ig, decay, _, st, lens = inputs(2000, 5, 128, T[ty], 3, state=True, ragged=True)
    decay = decay - 4                                  # 8 softplus(decay) below 0.34
    decay[D:] = 2.0 if far else -6.0
    args = cuda(x, rg, ig, decay)
    st, lens = cuda(st, lens)
    y, h = G.m3_gated_scan_with_state(*args, state=st, lengths=lens)
    cut = [t[..., :D].contiguous() for t in (*args, st)]
    y1, h1 = G.m3_gated_scan_with_state(*cut[:4], state=cut[4], lengths=lens)
    assert torch.equal(y1, y[..., :D]) and torch.equal(h1, h[:, :D])
