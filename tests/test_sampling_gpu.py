"""m3_sample against the definition in 64 bits (seq_oracle.kept_weights)."""

import numpy as np
import pytest
import torch

import seq_oracle as O
from redpanda_b200.sampling import m3_sample

pytestmark = pytest.mark.gpu
T = {"f32": torch.float32, "bf16": torch.bfloat16}


def _expect(logits, u, T_, k, p, m):
    """Tokens, and u with the numbers that lie on a border (closer than 1e-9)
    replaced before the kernel sees them."""
    rows = logits.shape[0]
    x = logits.double().numpy()
    per = [np.broadcast_to(np.asarray(v, dtype=np.float64), rows) for v in (T_, k, p, m)]
    u = u.clone()
    want = []
    for r in range(rows):
        w = O.kept_weights(x[r], per[0][r], int(per[1][r]), per[2][r], per[3][r])
        token, gap = O.draw(w, float(u[r]))
        while gap < 1e-9:
            u[r] = (float(u[r]) * 0.7 + 0.123) % 1.0
            token, gap = O.draw(w, float(u[r]))
        want.append(token)
    return torch.tensor(want), u


def _check(logits, u, T_=1.0, k=0, p=1.0, m=0.0):
    f = lambda v, t: torch.tensor(v, dtype=t).cuda() if isinstance(v, (list, np.ndarray)) else v  # noqa: E731
    # settings that the kernel holds in float32 are float32 in the oracle too
    r32 = lambda v: np.asarray(v, dtype=np.float32).astype(np.float64)  # noqa: E731
    want, u = _expect(logits, u, r32(T_), k, r32(p), r32(m))
    got = m3_sample(logits.cuda(), u.cuda(), f(T_, torch.float32), f(k, torch.int32),
                    f(p, torch.float32), f(m, torch.float32))
    assert got.dtype == torch.int64
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [1, 2, 31, 100, 1000, 8192, 40000])
@pytest.mark.parametrize("kw", [dict(), dict(k=5), dict(p=0.8), dict(m=0.1),
                                dict(T_=0.6, k=40, p=0.9, m=0.02), dict(T_=1.7, k=1),
                                dict(p=0.0), dict(p=0.999, T_=3.0), dict(T_=0.0), dict(m=1.0)])
def test_sample_matches_definition(V, kw, dtype):
    g = torch.Generator().manual_seed(V)
    rows = 24 if V < 8192 else 4
    logits = (torch.randn(rows, V, generator=g) * 2.5).to(T[dtype])
    _check(logits, torch.rand(rows, generator=g), **kw)


@pytest.mark.parametrize("kw", [dict(k=3), dict(k=7, p=0.5), dict(p=0.4), dict(p=0.75, k=6),
                                dict(k=2, m=0.5), dict()])
def test_sample_ties_go_to_the_lowest_index(kw):
    """Few distinct values: cuts fall inside ties."""
    g = torch.Generator().manual_seed(3)
    logits = torch.randint(0, 3, (64, 333), generator=g).float()
    logits[0] = 1.0                       # all equal
    logits[1, :] = -0.0
    logits[1, ::2] = 0.0                  # zeros of both signs are equal
    _check(logits, torch.rand(64, generator=g), **kw)


def test_sample_masks_and_odd_values():
    inf, nan, low = float("inf"), float("nan"), torch.finfo(torch.float32).min
    rows = [[-inf] * 6, [nan] * 6, [nan, -inf, 2.0, -inf, nan, nan], [low] * 6,
            [low, 0, low, 0, low, low], [inf, 1, inf, 2, 3, inf], [-inf, inf, 0, nan, 1, 2],
            [low, low, -inf, -inf, low, nan], [3e38, -3e38, 3e38, 0, 1, 2], [-inf, -3, -inf] * 2]
    logits = torch.tensor(rows)
    g = torch.Generator().manual_seed(1)
    for kw in (dict(), dict(k=2), dict(p=0.5), dict(m=0.3), dict(T_=0.0), dict(T_=1e-30),
               dict(T_=1e30, k=4)):
        for _ in range(4):
            _check(logits, torch.rand(len(rows), generator=g), **kw)
    got = m3_sample(logits.cuda(), torch.rand(len(rows)).cuda())
    assert got[:2].tolist() == [-1, -1]


def test_sample_border_numbers():
    """u = 0 takes the first kept token, u just below 1 (and 1) the last."""
    logits = torch.tensor([[-float("inf"), 0.0, 1.0, 0.5, -float("inf")]]).cuda()
    for u, want in ((0.0, 1), (float(np.nextafter(np.float32(1), 0)), 3), (1.0, 3)):
        assert m3_sample(logits, torch.tensor([u]).cuda()).item() == want


def test_sample_settings_per_row():
    g = torch.Generator().manual_seed(11)
    rows, V = 50, 777
    logits = torch.randn(rows, V, generator=g) * 3
    logits[torch.rand(rows, V, generator=g) < 0.5] = -float("inf")
    r = np.random.RandomState(2)
    T_ = r.uniform(0.0, 2.0, rows)
    T_[:5] = [0.0, -1.0, 0.1, 5.0, 1.0]
    k = r.randint(-1, 60, rows)
    _check(logits, torch.rand(rows, generator=g), T_, k, r.uniform(0, 1.2, rows),
           r.uniform(0, 0.3, rows))


def test_sample_strides_and_single_rows():
    g = torch.Generator().manual_seed(5)
    base = torch.randn(6, 500, generator=g).cuda()
    u = torch.rand(6, generator=g).cuda()
    a = m3_sample(base[:, 3:403], u, top_k=20)
    assert torch.equal(a, m3_sample(base[:, 3:403].contiguous(), u, top_k=20))
    assert torch.equal(m3_sample(base[:, :400].t().contiguous().t(), u),
                       m3_sample(base[:, :400].contiguous(), u))
    one = m3_sample(base[2], u[2])
    assert one.dim() == 0 and one == m3_sample(base, u)[2]
    assert torch.equal(m3_sample(base[:1].expand(6, 500), u),
                       m3_sample(base[:1].expand(6, 500).contiguous(), u))
    assert m3_sample(base[:0], u[:0]).shape == (0,)


def test_sample_large_vocabulary():
    g = torch.Generator().manual_seed(6)
    logits = torch.randn(2, 262144, generator=g)
    for kw in (dict(), dict(k=1000), dict(p=0.7), dict(p=0.9, m=0.01)):
        _check(logits, torch.rand(2, generator=g), **kw)


def test_sample_distribution():
    """The empirical distribution over a grid of u is the kept distribution:
    with u at n midpoints every token is drawn w n +- 1 times."""
    g = torch.Generator().manual_seed(7)
    x = torch.randn(50, generator=g)
    n = 4096
    u = ((torch.arange(n) + 0.5) / n).float()
    got = m3_sample(x.expand(n, 50).cuda(), u.cuda(), top_k=20, top_p=0.9).cpu()
    w = O.kept_weights(x.numpy(), 1.0, 20, float(np.float32(0.9)), 0.0)
    count = torch.bincount(got, minlength=50).double().numpy()
    assert (np.abs(count - w / w.sum() * n) <= 1).all()


def test_sample_is_capturable():
    x, u = torch.randn(8, 8192, device="cuda"), torch.rand(8, device="cuda")
    ref = m3_sample(x, u, top_k=50, top_p=0.9)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m3_sample(x, u, top_k=50, top_p=0.9)
    graph.replay()
    assert torch.equal(out, ref)


@pytest.mark.parametrize("V", [300, 8192, 40000])
@pytest.mark.parametrize("kw", [dict(m=0.02), dict(p=0.9, m=0.001), dict(p=0.3), dict(p=0.99),
                                dict(p=0.6, m=0.2), dict(p=1e-6), dict(m=1e-9)])
def test_sample_borders_among_many_and_few_tokens(V, kw):
    """Rows from peaked to flat, masked ones and ones with ties: the borders lie
    within the first tokens of the order, behind them, or in a long tie."""
    g = torch.Generator().manual_seed(V + 1)
    rows = 12
    logits = torch.randn(rows, V, generator=g) * torch.tensor(
        [0.0, 0.01, 0.3, 1, 2, 3, 5, 8, 20, 3, 3, 1])[:, None]
    logits[9] = logits[9].round()
    logits[10] = (logits[10] * 2).round() / 2
    logits[11][torch.rand(V, generator=g) < 0.97] = -float("inf")
    T_ = np.random.RandomState(V).uniform(0.5, 1.6, rows)
    _check(logits, torch.rand(rows, generator=g), T_, 0, kw.get("p", 1.0), kw.get("m", 0.0))


def test_sample_border_on_a_token():
    """top_p at, and a rounding beside, the cumulative weight of a token: decided
    as the 64-bit definition decides it (equal weights make the sums exact)."""
    V = 512
    logits = torch.zeros(1, V)
    for count in (1, 2, 128, 256, 511):
        for p in (count / V, np.nextafter(np.float32(count / V), np.float32(2)),
                  np.nextafter(np.float32(count / V), np.float32(0))):
            p = float(np.float32(p))
            w = O.kept_weights(logits[0].numpy(), 1.0, 0, p, 0.0)
            last = int(np.nonzero(w)[0][-1])
            got = m3_sample(logits.cuda(), torch.tensor([1.0]).cuda(), top_p=p)
            assert got.item() == last


def test_sample_from_threads_with_different_lengths():
    """Row lengths that need different amounts of shared memory, side by side."""
    from concurrent.futures import ThreadPoolExecutor
    g = torch.Generator().manual_seed(41)
    work = [(torch.randn(3, V, generator=g).cuda(), torch.rand(3, generator=g).cuda())
            for V in (12000, 32768, 5000, 30000, 16000, 25000)]

    def run(w):
        with torch.cuda.stream(torch.cuda.Stream()):
            out = [m3_sample(*w, top_k=40, top_p=0.9) for _ in range(20)]
            torch.cuda.current_stream().synchronize()
        return torch.stack(out)
    torch.cuda.synchronize()
    with ThreadPoolExecutor(len(work)) as pool:
        got = list(pool.map(run, work))
    for w, o in zip(work, got):
        assert (o == m3_sample(*w, top_k=40, top_p=0.9)).all()


def test_sample_top_k_of_other_integer_types():
    """Counts past 32 bits keep every token, negative ones too; none wraps."""
    g = torch.Generator().manual_seed(42)
    x, u = torch.randn(4, 100, generator=g).cuda(), torch.rand(4, generator=g).cuda()
    want = m3_sample(x, u, top_k=torch.tensor([0, 0, 3, 0], dtype=torch.int32).cuda())
    got = m3_sample(x, u, top_k=torch.tensor([2 ** 32 + 1, -2 ** 32 + 1, 3, 2 ** 40]).cuda())
    assert torch.equal(got, want)
    assert torch.equal(m3_sample(x, u, top_k=torch.tensor([0, 0, 3, 0], dtype=torch.uint8).cuda()),
                       want)
