"""The gated linear recurrence against its definition in 64 bits."""

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
