"""The sequence-model operators as they are used together: a selective layer
over a prompt and token by token, its training step, and lines of moves drawn
by the search model."""

import pytest
import torch
import torch.nn.functional as F

import seq_oracle as O
from redpanda_b200 import norm as N
from redpanda_b200 import selective as S
from redpanda_b200.mamba import Mamba, MambaConfig, RMSNorm
from redpanda_b200.sampling import m3_sample
from redpanda_b200.search_mamba import SearchMamba, SearchMambaConfig

pytestmark = pytest.mark.gpu


class Layer:
    """norm -> in_proj -> conv -> x_proj, dt_proj -> scan -> out_proj + residual -> head."""

    def __init__(self, d, n, k, r, vocab, seed):
        g = torch.Generator().manual_seed(seed)
        di = 2 * d
        rnd = lambda *s, c=1.0: torch.randn(*s, generator=g) * c  # noqa: E731
        self.p = dict(nw=1 + rnd(d, c=0.1), win=rnd(2 * di, d, c=d ** -0.5),
                      cw=rnd(di, k, c=k ** -0.5), cb=rnd(di, c=0.1),
                      wx=rnd(r + 2 * n, di, c=di ** -0.5), wdt=rnd(di, r, c=r ** -0.5),
                      db=torch.rand(di, generator=g) * 2 - 4,
                      A=-torch.arange(1.0, n + 1).repeat(di, 1), D=1 + rnd(di, c=0.1),
                      wout=rnd(d, di, c=di ** -0.5), fw=1 + rnd(d, c=0.1), fb=rnd(d, c=0.1),
                      head=rnd(vocab, d, c=3 * d ** -0.5))
        self.di, self.n, self.r, self.k = di, n, r, k

    def cuda(self):
        self.p = {k: v.cuda() for k, v in self.p.items()}
        return self

    def pre(self, x):
        p = self.p
        xz = F.linear(N.m3_rms_norm(x, p["nw"]), p["win"])
        return xz[..., :self.di], xz[..., self.di:]

    def inputs(self, u):
        p = self.p
        xd = F.linear(u, p["wx"])
        n, r = self.n, self.r
        return F.linear(xd[..., :r], p["wdt"]), xd[..., r:r + n], xd[..., r + n:]

    def post(self, x, y):
        p = self.p
        h = x + F.linear(y, p["wout"])
        return F.linear(N.m3_layer_norm(h, p["fw"], p["fb"]), p["head"])

    def prompt(self, x, lengths=None):
        p = self.p
        xb, z = self.pre(x)
        u, cs = S.m3_causal_conv_with_state(xb, p["cw"], p["cb"], lengths=lengths)
        dt, Bm, Cm = self.inputs(u)
        y, h = S.m3_selective_scan_with_state(u, dt, p["A"], Bm, Cm, D=p["D"], z=z,
                                              dt_bias=p["db"], lengths=lengths)
        return self.post(x, y), (cs, h)

    def token(self, x, state):
        p = self.p
        xb, z = self.pre(x)
        u = S.m3_causal_conv_step_(state[0], xb, p["cw"], p["cb"])
        dt, Bm, Cm = self.inputs(u)
        y = S.m3_selective_step_(state[1], u, dt, p["A"], Bm, Cm, D=p["D"], z=z, dt_bias=p["db"])
        return self.post(x, y)

    def plain(self, x):
        """The same in 64 bits on the CPU (one row)."""
        p = {k: v.detach().cpu().double() for k, v in self.p.items()}
        x = x.detach().cpu().double()
        B, L, d = x.shape
        xz = O.norm(x.reshape(-1, d), p["nw"], None, 1e-5, True).view(B, L, d) @ p["win"].T
        xb, z = xz[..., :self.di], xz[..., self.di:]
        u = O.conv(xb, p["cw"], p["cb"], True, None, None)[0]
        xd = u @ p["wx"].T
        n, r = self.n, self.r
        y = O.scan(u, xd[..., :r] @ p["wdt"].T, p["A"], xd[..., r:r + n], xd[..., r + n:], D=p["D"],
                   z=z, dt_bias=p["db"])["y"]
        h = x + y @ p["wout"].T
        return O.norm(h.reshape(-1, d), p["fw"], p["fb"], 1e-5, False).view(B, L, d) @ p["head"].T


@pytest.fixture(autouse=True)
def _no_tf32():
    old = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    yield
    torch.backends.cuda.matmul.allow_tf32 = old


def test_prompt_then_tokens_then_drawing():
    """A ragged batch of prompts, then tokens: logits of the whole sequence in
    64 bits, and the tokens drawn from them.

    Bar: a layer is about 20 chained roundings on top of the 30-step scan's 300
    and sums of up to 64 products in each projection: under 2000 e = 1.2e-4 of the
    largest logit; measured quantities add as square roots, so 2e-5 stands."""
    torch.manual_seed(0)
    layer = Layer(32, 16, 4, 4, 50, seed=1).cuda()
    lens = torch.tensor([21, 1, 0, 12], dtype=torch.int32)
    seqs = [torch.randn(1, int(n) + 6, 32) for n in lens]
    x = torch.zeros(4, 21, 32)
    for i, n in enumerate(lens):
        x[i, :n] = seqs[i][0, :n]
    with torch.no_grad():
        logits, state = layer.prompt(x.cuda(), lens.cuda())
        steps = [layer.token(torch.cat([s[:, n + t] for s, n in zip(seqs, lens.tolist())]).cuda(),
                             state) for t in range(6)]
    u = torch.rand(4, 6)
    for i, n in enumerate(lens.tolist()):
        ref = layer.plain(seqs[i])[0]
        got = torch.cat([logits[i, :n], torch.stack([s[i] for s in steps])]).cpu().double()
        assert (got - ref).abs().max() <= 2e-5 * ref.abs().max()
    for t in range(6):
        tok = m3_sample(steps[t], u[:, t].contiguous().cuda(), temperature=0.7, top_k=10, top_p=0.9)
        for i in range(4):
            w = O.kept_weights(steps[t][i].cpu().numpy(), float(torch.tensor(0.7)), 10,
                               float(torch.tensor(0.9)), 0.0)
            want, gap = O.draw(w, float(u[i, t]))
            assert gap < 1e-9 or tok[i].item() == want


def test_training_step_against_differences():
    """The layer's gradients: the loss along a random direction of every
    parameter, by differences of the 64-bit layer."""
    layer = Layer(16, 8, 4, 2, 20, seed=3)
    g = torch.Generator().manual_seed(4)
    x, wl = torch.randn(2, 19, 16, generator=g), torch.randn(2, 19, 20, generator=g)
    base = {k: v.clone() for k, v in layer.p.items()}
    layer.cuda()
    for v in layer.p.values():
        v.requires_grad_(True)
    xc = x.cuda().requires_grad_(True)
    out = layer.prompt(xc)[0]
    names = list(layer.p)
    grads = torch.autograd.grad((out * wl.cuda()).sum(), [layer.p[k] for k in names] + [xc])
    for k, gr in zip(names + ["x"], grads):
        v = torch.randn((x if k == "x" else base[k]).shape, generator=g).double()
        f = []
        for s in (1, -1):
            layer.p = {n: t.double() for n, t in base.items()}
            xx = x.double()
            if k == "x":
                xx = xx + s * 1e-4 * v
            else:
                layer.p[k] = layer.p[k] + s * 1e-4 * v
            f.append((layer.plain(xx) * wl.double()).sum().item())
        ours = gr.cpu().double() * v
        # 3e-5: the differences' h^2 terms and 2000 e / sqrt of the chain, as above
        assert abs((f[0] - f[1]) / 2e-4 - ours.sum().item()) <= 3e-5 * ours.abs().sum().item(), k


def _search(**kw):
    torch.manual_seed(0)
    cfg = SearchMambaConfig(d_model=64, n_layer=2, d_state=16, n_track_state=4, mimo_p=2,
                            vocab_size=96, **kw)
    return SearchMamba(cfg, eval_dim=32).cuda().eval()


def test_sample_lines_draws_from_the_continuation_head():
    """Moves and values against eager steps of the same model; the number that
    decides a move may not lie on a border of the eager distribution."""
    m = _search()
    board = torch.randint(0, 96, (12,), device="cuda")
    u = torch.rand(5, 7, generator=torch.Generator().manual_seed(2))
    moves, values = m.sample_lines(board, u.cuda(), temperature=0.9, top_k=20, top_p=0.95)
    assert moves.shape == (5, 7) and values.shape == (5,) and (moves >= 0).all()
    with torch.no_grad():
        for i in range(5):
            hidden, cache = m.prime_board(board)
            for t in range(7):
                logits = m.continuation_head(hidden)[0].cpu().numpy()
                w = O.kept_weights(logits, float(torch.tensor(0.9)), 20, float(torch.tensor(0.95)),
                                   0.0)
                want, gap = O.draw(w, float(u[i, t]))
                assert gap < 1e-4 or moves[i, t].item() == want
                hidden, cache = m.backbone.step(moves[i:i + 1, t], cache)
            ref = torch.tanh(m.value_head(hidden)).item()
            assert abs(values[i].item() - ref) <= 2e-5
    again = m.sample_lines(board, u.cuda(), temperature=0.9, top_k=20, top_p=0.95)
    assert torch.equal(moves, again[0]) and torch.equal(values, again[1])
    per = m.sample_lines(board, u.cuda(), temperature=torch.full((5,), 0.9, device="cuda"),
                         top_k=torch.full((5,), 20, device="cuda", dtype=torch.int32),
                         top_p=torch.full((5,), 0.95, device="cuda"))
    assert torch.equal(moves, per[0])
    with pytest.raises(ValueError):
        m.sample_lines(board, u[0].cuda())


def test_model_norms_on_the_kernels():
    """RMSNorm.use_kernel and LayerNorm.use_kernel: the model's outputs and
    gradients up to rounding; off, they are torch's bits."""
    torch.manual_seed(1)
    cfg = MambaConfig(d_model=64, n_layer=2, d_state=16, n_track_state=4, mimo_p=2, vocab_size=96)
    m = Mamba(cfg).cuda()
    ids = torch.randint(0, 96, (3, 20), device="cuda")

    def run():
        m.zero_grad()
        y = m(ids)
        y.pow(2).mean().backward()
        return [y.detach()] + [p.grad.clone() for p in m.parameters()]
    off = run()
    assert all(torch.equal(a, b) for a, b in zip(off, run()))
    RMSNorm.use_kernel = True
    try:
        on = run()
        with torch.no_grad():
            assert (m(ids) - on[0]).abs().max() <= 5e-6 * on[0].abs().max()
    finally:
        RMSNorm.use_kernel = False
    # the bars of the model's own parity tests: 5e-6 forward, 5e-5 gradients
    for i, (a, b) in enumerate(zip(off, on)):
        assert (a - b).abs().max() <= (5e-6 if i == 0 else 5e-5) * a.abs().max()
    s = _search()
    board = torch.randint(0, 96, (12,), device="cuda")
    seqs = torch.randint(0, 96, (4, 5), device="cuda")
    with torch.no_grad():
        ref = s.evaluate_with_continuation(board, seqs)
        N.LayerNorm.use_kernel = True
        try:
            got = s.evaluate_with_continuation(board, seqs)
        finally:
            N.LayerNorm.use_kernel = False
    for a, b in zip(ref, got):
        assert (a - b).abs().max() <= 5e-6 * max(1.0, a.abs().max().item())


def test_sample_lines_needs_a_line_and_a_move():
    m = _search()
    board = torch.randint(0, 96, (12,), device="cuda")
    for shape in ((0, 3), (3, 0), (3,)):
        with pytest.raises(ValueError):
            m.sample_lines(board, torch.zeros(shape, device="cuda"))
