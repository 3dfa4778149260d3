"""m3_sample where its ways of deciding a row meet: rows without any cut, settings
that are not numbers, borders in large vocabularies."""

import numpy as np
import pytest
import torch

import seq_oracle as O
from redpanda_b200.sampling import m3_sample
from test_sampling_gpu import T, _check

pytestmark = pytest.mark.gpu


def _overwrite_shared_memory():
    """Products whose tiles fill the SMs' shared memory with other bits."""
    for dtype in (torch.float32, torch.bfloat16):
        a = torch.full((2048, 2048), 1e30, device="cuda", dtype=dtype)
        a @ a


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,V", [(24, 257), (24, 1000), (600, 300), (4, 8192), (3, 40000)])
def test_sample_without_cuts_sets_up_its_own_tables(rows, V, dtype):
    """The default settings: no cut stands between the row's maximum and the draw,
    and nothing that an earlier kernel left in shared memory takes part."""
    g = torch.Generator().manual_seed(V + rows)
    logits = (torch.randn(rows, V, generator=g) * 2.5).to(T[dtype])
    for kw in (dict(), dict(T_=0.7), dict(k=V + 5)):
        _overwrite_shared_memory()
        _check(logits, torch.rand(rows, generator=g), **kw)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [7, 255, 256, 257, 700, 1024, 1025, 8192, 40000])
def test_sample_top_p_that_is_no_number_takes_the_first_token(V, dtype):
    """top_p of NaN, or below 0, per row counts as 0, whatever the number of
    candidates and the other settings: the first token of the order."""
    g = torch.Generator().manual_seed(V)
    rows = 6
    logits = (torch.randn(rows, V, generator=g) * 0.5).to(T[dtype])
    logits[1] = 0.25                       # ties: the lowest index
    logits[2, :V // 2] = -float("inf")
    most = logits.float() == logits.float().max(1, keepdim=True).values
    want = torch.where(most, torch.arange(V), V).min(1).values
    assert want[1] == 0
    x, u = logits.cuda(), torch.full((rows,), 0.999).cuda()
    for bad in (float("nan"), -0.5, -float("inf"), 0.0):
        p = torch.full((rows,), bad).cuda()
        for kw in (dict(), dict(top_k=3), dict(top_k=V - 1), dict(min_p=1e-4), dict(min_p=0.3),
                   dict(temperature=0.5), dict(temperature=50.0, min_p=0.01)):
            got = m3_sample(x, u, top_p=p, **kw)
            assert torch.equal(got.cpu(), want), (bad, kw)
    # beside rows with a top_p of their own, whose draws stay theirs
    p = torch.tensor([0.5, float("nan")] * 3).cuda()
    ref = m3_sample(x, u, top_p=0.5, min_p=1e-4)
    got = m3_sample(x, u, top_p=p, min_p=1e-4).cpu()
    assert torch.equal(got[::2], ref[::2].cpu()) and torch.equal(got[1::2], want[1::2])


@pytest.mark.parametrize("V,rows", [(262144, 1), (262144, 5), (32768, 1), (32768, 400), (4100, 3)])
@pytest.mark.parametrize("T_", [1.0, 0.7])
def test_sample_top_p_border_beside_a_token_before_a_long_tail(V, rows, T_):
    """top_p a little below and above the share of a prefix: 600 tokens of falling
    weight before a tail of equal weights that are no power of two, whose fp32 sum
    rounds one way.  u = 1 draws the last kept token, as the 64-bit definition
    counts them."""
    heads = 600
    x = torch.full((V,), float(np.log(0.7) - np.log(V - heads) + np.log(heads)))
    x[:heads] = -torch.arange(heads) * 1e-3
    x = x * T_
    w = O.kept_weights(x.numpy(), float(np.float32(T_)), 0, 1.0, 0.0)
    cum = np.cumsum(w[:heads]) / w.sum()
    ps, want = [], []
    for j in (0, 1, 99, 300, 599):
        for off in (-1e-4, -3e-5, -1e-5, -2e-6, -2e-7, 2e-7, 2e-6, 1e-5, 3e-5, 1e-4):
            p = float(np.float32(cum[j] * (1 + off)))
            kept = O.kept_weights(x.numpy(), float(np.float32(T_)), 0, p, 0.0)
            ps.append(p)
            want.append(int(np.nonzero(kept)[0][-1]))
    logits = x.cuda()
    for p, n in zip(ps, want):
        got = m3_sample(logits.expand(rows, V), torch.ones(rows).cuda(), temperature=T_, top_p=p)
        assert (got == n).all(), (p, n, got)


@pytest.fixture
def _no_waiting():
    torch.cuda.set_sync_debug_mode("error")
    yield
    torch.cuda.set_sync_debug_mode("default")


@pytest.mark.parametrize("shape", [(5, 900), (900,), (0, 900)])
def test_sample_settings_of_one_number_on_the_gpu(shape, _no_waiting):
    """0-dim tensors on the GPU: the draw of the same numbers, without a wait for
    the GPU, and so in a captured graph, where a later value takes part."""
    g = torch.Generator("cuda").manual_seed(9)
    x = torch.randn(shape, device="cuda", generator=g) * 2
    u = torch.rand(shape[:-1], device="cuda", generator=g)
    new = lambda v, t: torch.full((), v, device="cuda", dtype=t)  # noqa: E731
    kw = dict(temperature=new(0.75, torch.float64), top_k=new(30, torch.int64),
              top_p=new(0.875, torch.float32), min_p=new(0.015625, torch.bfloat16))
    ref = m3_sample(x, u, temperature=0.75, top_k=30, top_p=0.875, min_p=0.015625)
    got = m3_sample(x, u, **kw)
    assert got.shape == ref.shape == u.shape
    torch.cuda.set_sync_debug_mode("default")
    assert torch.equal(got, ref)
    if x.numel() == 0:
        return
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m3_sample(x, u, **kw)
    graph.replay()
    assert torch.equal(out, ref)
    kw["top_k"].fill_(1)
    graph.replay()
    assert torch.equal(out, x.argmax(-1))
