"""The operators of a gated recurrent layer in 64 bits on the CPU, straight from
their definitions, with bounds for the rounding of an fp32 evaluation.

``gated`` carries the bound along with the recurrence (first-order running error
analysis, e = 2^-24).  With l = -c softplus(decay) r, r = sigmoid(rg):

* r: (1.3 |rg| + 10) e (the MUFU unit's 2^x and reciprocal, the argument rounded
  once); softplus, the two products and c: 8 e more; so l has lam e,
  lam = 1.3 |rg| + 18, relative.
* a = e^l: lam |l| e from l, 2 e of its own (polynomial and final sum), and 3 e
  per step for the products and sums of the runs that are joined.
* m = sqrt(-p (2 + p)), p = e^l - 1: l's error counts at most once in p (l e^l /
  (e^l - 1) <= 1), p's own 2 e and the product 2 e; half of these through the
  root; the root's MUFU form and product 3 e.
* i: (1.3 |ig| + 10) e.
* From l = -87 down (e^l = 1.6e-38, where fp32 ends) the kernel's a is 0: an error of
  all of a, relative 1 (l itself off by lam e: from -87 (1 - lam e)).
"""

import torch

from seq_oracle import E, _lens, half_step, softplus  # noqa: F401


def gated(x, rg, ig, decay, c=8.0, state=None, lengths=None, g=None):
    """Dict of y, h and, with g, dx, drg, dig, ddecay; and of their bounds under
    the names with "+" in front."""
    x, rg, ig, decay = (t.double() for t in (x, rg, ig, decay))
    B, L, D = x.shape
    r, i = torch.sigmoid(rg), torch.sigmoid(ig)
    l = -c * softplus(decay) * r
    a, m = torch.exp(l), torch.sqrt(-torch.expm1(2 * l))
    lam = 1.3 * rg.abs() + 18
    gone = l <= -87 * (1 - lam * E)
    ea = torch.where(gone, 1.0, (lam * l.abs() + 5) * E)   # relative error of a
    em = (lam / 2 + 5) * E                           # of m
    ei = (1.3 * ig.abs() + 10) * E
    b = m * i * x
    eb = (em + ei + 2 * E) * b.abs()                 # absolute
    live = torch.tensor([[t < n for t in range(L)] for n in _lens(lengths, B, L)],
                        dtype=torch.bool).view(B, L, 1)
    h = torch.zeros(B, D, dtype=torch.float64) if state is None else state.double()
    eh = torch.zeros_like(h)
    y, ey, before, ebefore = (torch.zeros_like(x) for _ in range(4))
    for t in range(L):
        before[:, t], ebefore[:, t] = h, eh
        new = a[:, t] * h + b[:, t]
        enew = a[:, t] * (eh + h.abs() * ea[:, t]) + eb[:, t] + 2 * E * new.abs()
        h, eh = torch.where(live[:, t], new, h), torch.where(live[:, t], enew, eh)
        y[:, t], ey[:, t] = torch.where(live[:, t], new, 0), torch.where(live[:, t], enew, 0)
    out = {"y": y, "+y": ey, "h": h, "+h": eh}
    if g is None:
        return out
    g = torch.where(live, g.double(), 0)
    q, eq = torch.zeros_like(x), torch.zeros_like(x)
    v = ev = torch.zeros(B, D, dtype=torch.float64)
    for t in range(L - 1, -1, -1):
        q[:, t] = g[:, t] + v
        eq[:, t] = ev + 2 * E * q[:, t].abs()
        at = torch.where(live[:, t], a[:, t], 1.0)
        v, ev = at * q[:, t], at * (eq[:, t] + q[:, t].abs() * ea[:, t])
    q, eq = torch.where(live, q, 0), torch.where(live, eq, 0)
    inv = torch.where(m > 0, 1 / m, torch.zeros_like(m))
    ux = i * x
    A = l * (a * before - a * a * inv * ux)
    eA = l.abs() * (a * ebefore + a * before.abs() * (ea + 2 * E)
                    + a * a * inv * ux.abs() * (2 * ea + em + ei + 5 * E)) \
        + A.abs() * (lam + 3) * E
    R, eR = 1 - r, r * lam * E + E
    e, ee = q * A, q.abs() * eA + eq * A.abs() + (q * A).abs() * E
    out.update({"dx": q * m * i, "+dx": eq * m * i + (q * m * i).abs() * (em + ei + 3 * E),
                "drg": e * R, "+drg": ee * R + e.abs() * eR + (e * R).abs() * E})
    dig = q * m * x * i * (1 - i)
    mix = (m * x * i).abs()
    out.update({"dig": dig, "+dig": eq * mix * (1 - i) + (em + ei + 4 * E) * dig.abs()
                + q.abs() * mix * (i * ei + E)})
    sp = softplus(decay)
    ratio = torch.where(sp > 0, torch.sigmoid(decay) / sp, torch.ones_like(sp))
    # partial sums: 8 steps, a thread's passes, warps, CTAs; one rounding each at most
    terms = B * L / 8 + 64
    total = e.sum((0, 1)) * ratio
    out.update({"ddecay": total, "+ddecay": ratio * (ee.sum((0, 1))
                                                     + terms * E * e.abs().sum((0, 1)))
                + 12 * E * total.abs()})
    return out


def excess(got, ref, bound, dtype):
    """Largest |got - ref| over what rounding allows (at most 1 when in bounds)."""
    got = got.detach().cpu().double()
    tiny = torch.finfo(torch.float32).tiny * 4       # flushed to zero
    tol = bound * 1.01 + half_step(dtype) * (ref.abs() + bound) + tiny
    return float(((got - ref).abs() / tol).max()) if ref.numel() else 0.0
