"""The scan's backward over batches whose partials do not fit one buffer."""

import pytest
import torch

from redpanda_b200 import _lib
from redpanda_b200 import selective as S

pytestmark = pytest.mark.gpu
E = 2.0 ** -24


def _workspace(B, L, D, N, dtype=0):
    return _lib.load().m3_selective_bwd_workspace_bytes(_lib.SelDesc(B, L, D, N, dtype, 1))


def test_backward_workspace_is_bounded_over_the_batch():
    """256 rows of 4096 steps, 1536 channels, 128 states: 103 GB of partials, taken
    in slabs of 2 GB; from there on more rows cost nothing but the time."""
    a, b = _workspace(256, 4096, 1536, 128), _workspace(4096, 4096, 1536, 128)
    assert 0 < a < 3 << 30 and b <= a
    assert _workspace(1 << 14, 4096, 1536, 16) < 3 << 30
    # a batch below the bound has one buffer for all of it
    assert _workspace(256, 64, 1536, 32) >= 256 * 64 * 48 * 2 * 32 * 4


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_backward_in_slabs_equals_the_parts(dtype):
    """Gradients of a batch in two slabs against those of its parts (one each):
    the rows' own bit for bit; the parameters' sums up to their additions.  All
    terms of those are positive (growing states of positive inputs), so a sum of
    B L terms in any order is off by at most (B L + 20 L + N + 64) e of itself, on
    each side: 20 roundings per step there and back, N and D sums, the ends."""
    B, L, D, N, cut = 1300, 33, 1024, 128, 701
    row = 64 * L * 2 * 128 * 4                       # 64 tiles of 16 channels
    assert cut * row <= 2 << 30 < B * row
    g = torch.Generator("cuda").manual_seed(3)
    pos = lambda *s, c=1.0: torch.rand(*s, device="cuda", generator=g) * c  # noqa: E731
    a = dict(u=pos(B, L, D).to(dtype), dt=pos(B, L, D, c=0.02).to(dtype), A=pos(D, N),
             Bm=pos(B, L, N).to(dtype), Cm=pos(B, L, N).to(dtype), D=pos(D),
             dt_bias=pos(D, c=0.01))
    n = torch.randint(0, L + 1, (B,), device="cuda", generator=g, dtype=torch.int32)
    n[::7], n[1::11] = L, 0
    h0, gr = pos(B, D, N), pos(B, L, D).to(dtype)

    def run(lo, hi):
        x = {k: (v[lo:hi] if v.shape[0] == B else v).detach().requires_grad_(True)
             for k, v in a.items()}
        y = S.m3_selective_scan(**x, softplus=False, state=h0[lo:hi], lengths=n[lo:hi])
        return dict(zip(x, torch.autograd.grad(y, list(x.values()), gr[lo:hi])))
    whole, one, two = run(0, B), run(0, cut), run(cut, B)
    tol = 2 * (B * L + 20 * L + N + 64) * E
    for k, v in whole.items():
        if v.shape[0] == B:
            assert torch.equal(v, torch.cat([one[k], two[k]])), k
        else:
            ref = one[k].double() + two[k].double()
            assert (ref > 0).all() and ((v.double() - ref).abs() <= tol * ref).all(), k


def test_backward_in_slabs_of_rows_that_are_split_along_time():
    """Two rows so long that each is a slab, their steps split over CTAs, against
    either row alone (another split).  All terms are positive (the step sizes'
    gradient is left out) and gates below e^-0.5 forget within 60 steps to 1e-13,
    so each side is off by at most (20 * 60 + N + 64) e beside the sums over D
    channels (dB, dC) and B L steps (the parameters)."""
    B, L, D, N = 2, 44000, 1536, 64
    assert 48 * L * 2 * 64 * 4 > 1 << 30
    assert _workspace(B, L, D, N, 1) < 3 << 30
    g = torch.Generator("cuda").manual_seed(5)
    pos = lambda *s: torch.rand(*s, device="cuda", generator=g)  # noqa: E731
    bf = torch.bfloat16
    a = dict(u=pos(B, L, D).to(bf), A=-1 - pos(D, N), Bm=pos(B, L, N).to(bf),
             Cm=pos(B, L, N).to(bf), D=pos(D))
    dt, gr = (0.5 + pos(B, L, D)).to(bf), pos(B, L, D).to(bf)
    n = torch.tensor([L, L - 1234], device="cuda", dtype=torch.int32)

    def run(lo, hi):
        x = {k: (v[lo:hi] if v.dim() == 3 else v).detach().requires_grad_(True)
             for k, v in a.items()}
        y = S.m3_selective_scan(dt=dt[lo:hi], **x, softplus=False, lengths=n[lo:hi])
        return dict(zip(x, torch.autograd.grad(y, list(x.values()), gr[lo:hi])))
    whole, rows = run(0, B), [run(i, i + 1) for i in range(B)]
    k, half = 20 * 60 + N + 64, 2.0 ** -8          # half a step of bf16, on each side
    for name, v in whole.items():
        if v.dim() == 3:
            tol = 2 * ((k + D) * E + half)
            for i in range(B):
                p, q = v[i].float(), rows[i][name][0].float()
                assert ((p - q).abs() <= tol * q).all(), name
                assert (q[:n[i]] > 0).all() and not q[n[i]:].any(), name
        else:
            ref = rows[0][name].double() + rows[1][name].double()
            assert ((v.double() - ref).abs() <= 2 * (k + B * L) * E * ref).all(), name
