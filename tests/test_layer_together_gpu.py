"""The operators of a gated recurrent layer as they are used together: a stack of
such layers over prompts, token by token with 4-bit weights, and its training
step; and inside the framework's own models."""

import copy

import pytest
import torch
import torch.nn.functional as F

import layer_oracle as O
import seq_oracle as SO
from redpanda_b200 import gated as G
from redpanda_b200 import norm as N
from redpanda_b200 import selective as S
from redpanda_b200.graphs import StepGraph
from redpanda_b200.mamba import Mamba, Mamba3Block, MambaConfig
from redpanda_b200.quant import Q4Weight, m3_rows_linear_q4

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_tf32():
    old = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    yield
    torch.backends.cuda.matmul.allow_tf32 = old


class Stack:
    """layers of: add + norm -> in_proj (x, two gates) -> conv -> recurrence -> out_proj."""

    def __init__(self, layers, d, k, seed):
        g = torch.Generator().manual_seed(seed)
        rnd = lambda *s, c=1.0: torch.randn(*s, generator=g) * c  # noqa: E731
        self.d, self.k, self.p, self.q = d, k, [], []
        for _ in range(layers):
            q = {n: Q4Weight.quantize(rnd(o, i, c=i ** -0.5), 32)
                 for n, o, i in (("win", 3 * d, d), ("wout", d, d))}
            self.q.append({n: w.to("cuda") for n, w in q.items()})
            p = dict(nw=1 + rnd(d, c=0.1), cw=rnd(d, k, c=k ** -0.5), cb=rnd(d, c=0.1),
                     decay=rnd(d) - 4, **{n: w.dequantize() for n, w in q.items()})
            self.p.append({n: t.cuda() for n, t in p.items()})

    def prompt(self, x, lengths=None):
        """Stream behind the layers, and the states."""
        branch, states = torch.zeros_like(x), []
        for p in self.p:
            h, x = N.m3_add_rms_norm(branch, x, p["nw"])
            u, a, b = F.linear(h, p["win"]).split(self.d, dim=-1)
            u, cs = S.m3_causal_conv_with_state(u, p["cw"], p["cb"], lengths=lengths)
            y, st = G.m3_gated_scan_with_state(u, a, b, p["decay"], lengths=lengths)
            branch = F.linear(y, p["wout"])
            states.append((cs, st))
        return x + branch, states

    def token(self, x, states):
        """One token per row (up to 8), the projections on 4-bit weights."""
        x = x.clone()
        for p, q, (cs, st) in zip(self.p, self.q, states):
            u, gates = m3_rows_linear_q4(x, q["win"], norm_weight=p["nw"], eps=1e-5, split=self.d)
            u = S.m3_causal_conv_step_(cs, u, p["cw"], p["cb"])
            y = G.m3_gated_step_(st, u, gates[:, :self.d], gates[:, self.d:], p["decay"])
            m3_rows_linear_q4(y, q["wout"], residual=x, out0=x)
        return x

    def plain(self, x):
        """The same in 64 bits on the CPU (one row)."""
        x = x.double().cpu()
        for p in self.p:
            p = {n: t.detach().cpu().double() for n, t in p.items()}
            h = SO.norm(x[0], p["nw"], None, 1e-5, True)[None]
            u, a, b = (h @ p["win"].T).split(self.d, dim=-1)
            u = SO.conv(u, p["cw"], p["cb"], True, None, None)[0]
            x = x + O.gated(u, a, b, p["decay"])["y"] @ p["wout"].T
        return x


def test_prompt_then_tokens_on_4_bit_weights():
    """A ragged batch of prompts, then tokens in lockstep, against the whole
    sequence in 64 bits.  Bar: two layers of about 40 chained roundings each, on
    the 30 steps' running error of the recurrence (5 e and 18 |l| e per step) and
    sums of up to 32 products per projection: under 1000 e = 6e-5 of the largest
    value; measured quantities add as square roots, so 1e-5 stands."""
    stack = Stack(2, 32, 4, seed=2)
    lens = torch.tensor([19, 1, 0, 11], dtype=torch.int32)
    g = torch.Generator().manual_seed(3)
    seqs = [torch.randn(1, int(n) + 5, 32, generator=g) for n in lens]
    x = torch.zeros(4, 19, 32)
    for i, n in enumerate(lens.tolist()):
        x[i, :n] = seqs[i][0, :n]
    with torch.no_grad():
        out, states = stack.prompt(x.cuda(), lens.cuda())
        steps = [stack.token(torch.cat([s[:, n + t] for s, n in zip(seqs, lens.tolist())]).cuda(),
                             states) for t in range(5)]
    for i, n in enumerate(lens.tolist()):
        ref = stack.plain(seqs[i])[0]
        got = torch.cat([out[i, :n], torch.stack([s[i] for s in steps])]).cpu().double()
        assert (got - ref).abs().max() <= 1e-5 * ref.abs().max()


def test_training_step_against_autograd_in_64_bits():
    """Gradients of every parameter through two layers; bar: 2e-5 of the largest
    gradient of each (about 300 chained roundings of 2^-24)."""
    stack = Stack(2, 16, 3, seed=5)
    x = torch.randn(3, 21, 16, generator=torch.Generator().manual_seed(1))
    up = torch.randn(3, 21, 16, generator=torch.Generator().manual_seed(2))
    leaves = [t.requires_grad_(True) for p in stack.p for t in p.values()]
    xs = x.cuda().requires_grad_(True)
    grads = torch.autograd.grad(stack.prompt(xs)[0], [xs, *leaves], up.cuda())
    ref_p = [{n: t.detach().cpu().double().requires_grad_(True) for n, t in p.items()}
             for p in stack.p]
    xd = x.double().requires_grad_(True)
    s = xd
    for p in ref_p:
        h = s * (s.square().mean(-1, keepdim=True) + 1e-5) ** -0.5 * p["nw"]
        u, a, b = (h @ p["win"].T).split(16, dim=-1)
        rows = torch.cat([u.new_zeros(3, 2, 16), u], 1)
        c = p["cb"] + sum(rows[:, k:k + 21] * p["cw"][:, k] for k in range(3))
        u = c * torch.sigmoid(c)
        l = -8 * F.softplus(p["decay"]) * torch.sigmoid(a)
        st, ys = u.new_zeros(3, 16), []
        for t in range(21):
            st = torch.exp(l[:, t]) * st + torch.sqrt(-torch.expm1(2 * l[:, t])) * \
                torch.sigmoid(b[:, t]) * u[:, t]
            ys.append(st)
        s = s + torch.stack(ys, 1) @ p["wout"].T
    refs = torch.autograd.grad(s, [xd, *(t for p in ref_p for t in p.values())], up.double())
    for ours, ref in zip(grads, refs):
        assert (ours.cpu().double() - ref).abs().max() <= 2e-5 * ref.abs().max()


def test_token_steps_in_a_captured_graph():
    """The token path replayed gives the eager path's bits, in its own state."""
    stack = Stack(2, 32, 4, seed=8)
    xs = torch.randn(6, 3, 32, generator=torch.Generator().manual_seed(9)).cuda()

    def fresh():
        return [(torch.zeros(3, 3, 32, device="cuda"), torch.zeros(3, 32, device="cuda"))
                for _ in stack.p]
    with torch.no_grad():
        eager, st = [], fresh()
        for x in xs:
            eager.append(stack.token(x, st))
        static, st2 = xs[0].clone(), fresh()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = stack.token(static, st2)
        for a in (t for pair in st2 for t in pair):
            a.zero_()
        for x, ref in zip(xs, eager):
            static.copy_(x)
            graph.replay()
            assert torch.equal(out, ref)


# ---------------------------------------------------------------- inside the models

def model(**kw):
    torch.manual_seed(0)
    cfg = MambaConfig(d_model=64, n_layer=3, vocab_size=40, d_state=32, mimo_p=2,
                      n_track_state=16, **kw)
    return Mamba(cfg).cuda()


@pytest.mark.parametrize("bf16", [False, True])
def test_model_with_the_fused_addition_and_norm(bf16):
    """Loss gradients of the same model with and without ``fuse_add_norm``: fp32
    within a few hundred roundings of 2^-24; in a bf16 layer the branches are bf16
    either way, and a norm's last fp32 bit can move a bf16 rounding (2^-8), which
    averages out over a gradient's sums: 2 % of its largest value."""
    m = model()
    ids = torch.randint(0, 40, (4, 17), generator=torch.Generator().manual_seed(4)).cuda()
    res = []
    for fused in (False, True):
        m.fuse_add_norm = fused
        m.zero_grad(set_to_none=True)
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=bf16):
            h = m(ids)
        assert h.dtype == torch.float32
        h.square().mean().backward()
        res.append([h.detach()] + [p.grad.clone() for p in m.parameters() if p.grad is not None])
    assert len(res[0]) == len(res[1])
    bar = 2e-2 if bf16 else 5e-5
    for a, b in zip(*res):
        assert (a - b).abs().max() <= bar * a.abs().max().clamp(min=1e-12)


def test_fused_addition_and_norm_is_off_where_it_does_not_apply():
    m = model()
    ids = torch.zeros(1, 3, dtype=torch.long, device="cuda")
    m.fuse_add_norm = True
    x = m.embedding(ids)
    assert m._add_norm_ok(x)
    with torch.no_grad():
        assert not m._add_norm_ok(x)
    m.grad_checkpoint = True
    assert not m._add_norm_ok(x)
    m.eval()
    assert m._add_norm_ok(x)
    with torch.autocast("cuda", dtype=torch.float16):
        assert not m._add_norm_ok(x)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert m._add_norm_ok(x)


def test_step_on_4_bit_weights():
    """The small-batch step with 4-bit projections is that of a model whose weights
    are what the codes stand for, eager and in a captured graph; other batches and
    the full weights stay as they were."""
    m = model()
    names = ("in_proj", "x_proj", "out_proj")
    full = copy.deepcopy(m)
    assert m.quantize_step_(group=32, names=names) is m
    stand_in = copy.deepcopy(full)
    with torch.no_grad():
        for a, b in zip(stand_in.layers, m.layers):
            for n in names:
                getattr(a["mixer"], n).weight.copy_(b["mixer"].step_q4[n][0].dequantize())
    ids = torch.randint(0, 40, (2, 9), generator=torch.Generator().manual_seed(4)).cuda()
    with torch.no_grad():
        _, cache = full.prime_cache(ids[:, :5])
        mine = lambda: [tuple(t.clone() for t in e) for e in cache]  # noqa: E731
        ca, cb = mine(), mine()
        graph = StepGraph(m, 2)
        graph.load_(mine())
        for t in range(5, 9):
            ha, _ = m.step_fused_(ids[:, t], ca)
            hb, _ = stand_in.step_fused_(ids[:, t], cb)
            # projections of 128 products and three layers: a few hundred roundings
            assert (ha - hb).abs().max() <= 5e-5 * hb.abs().max()
            assert torch.equal(graph.step(ids[:, t])[0], ha)
        # a batch past the small step's, and priming: the full weights' bits
        n = Mamba3Block.small_step_max_batch + 1
        wide = [(torch.zeros(n, 128, 32, device="cuda"), torch.zeros(n, 128, 32, device="cuda"))
                for _ in m.layers]
        again = copy.deepcopy(wide)
        tok = torch.arange(n, device="cuda")
        assert torch.equal(m.step_fused_(tok, wide)[0], full.step_fused_(tok, again)[0])
        assert torch.equal(m.prime_cache(ids)[0], full.prime_cache(ids)[0])
        # a changed weight is not stepped with its old codes
        m.layers[1]["mixer"].out_proj.weight.mul_(2)
        with pytest.raises(RuntimeError, match="quantize_step_"):
            m.step_fused_(ids[:, 0], mine())
        m.layers[1]["mixer"].out_proj.weight.mul_(0.5)
        m.quantize_step_(names=())
        held = graph.hidden.clone()
        graph.load_(cb)        # the graph has its own 4-bit weights
        ref = stand_in.step_fused_(ids[:, 0], [tuple(t.clone() for t in e) for e in cb])[0]
        assert (graph.step(ids[:, 0])[0] - ref).abs().max() <= 5e-5 * ref.abs().max()
        assert not torch.equal(held, graph.hidden)
        assert torch.equal(m.step_fused_(ids[:, 0], mine())[0],
                           full.step_fused_(ids[:, 0], mine())[0])
    assert set(m.state_dict()) == set(full.state_dict())
    with pytest.raises(ValueError):
        m.quantize_step_(names=("dt_proj",))


@pytest.mark.parametrize("autocast", [False, True])
def test_fused_addition_and_norm_of_a_narrow_stream(autocast):
    """bf16 embeddings: the stream gets the type of torch's sums, float32 behind the
    first layer of fp32 weights.  Against the same model unfused on the same norm
    kernels: fp32 within a few hundred roundings of 2^-24 (a stream held in bf16 is
    2^-9 = 2e-3 off); with a bf16 stream on both sides, or where a gradient is rounded
    to bf16 up to three times, as in the test above.  The loss is linear: the sum of an
    RMS norm's squares hardly depends on its row, and its gradients are differences."""
    m = model()
    for norm in m._norms():
        norm.use_kernel = True
    g = torch.Generator().manual_seed(6)
    emb = torch.randn(4, 17, 64, generator=g).bfloat16().cuda().requires_grad_(True)
    up = torch.randn(4, 17, 64, generator=g).cuda()
    res = []
    for fused in (False, True):
        m.fuse_add_norm = fused
        m.zero_grad(set_to_none=True)
        emb.grad = None
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
            assert m._add_norm_ok(emb) == fused
            h = m(None, input_embeds=emb)
        assert h.dtype == torch.float32
        (h * up).sum().backward()
        assert emb.grad.dtype == torch.bfloat16
        res.append([emb.grad.float(), h.detach()] + [p.grad.clone() for p in m.parameters()
                                                     if p.grad is not None])
    assert len(res[0]) == len(res[1])
    for i, (a, b) in enumerate(zip(*res)):
        bar = 2e-2 if autocast or i == 0 else 5e-5
        assert (a - b).abs().max() <= bar * a.abs().max().clamp(min=1e-12)
