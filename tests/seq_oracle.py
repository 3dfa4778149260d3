"""The sequence-model operators in 64 bits on the CPU, straight from their
definitions, with bounds for the rounding of an fp32 evaluation.

Bounds.  A computed sum of products of fp32 values, in which every path from an
input to the output passes at most k roundings of relative size e = 2^-24,
differs from the exact value by at most k e (to first order) times the sum of
the absolute values of its paths.  ``scan`` evaluates the same formulas with
absolute values for that sum (``magnitude=True``).  A step of the recurrence
costs a path: the gate (ex2.approx, 2 ulp = 4 e; the rounding of A log2(e), of
log2(e) itself and of the product, 3 e |de A| <= 3 e x with x e^-x <= 0.37 e; the
softplus of the step size, 4 e |de A|), and two roundings of the update: under
10 e.  A gradient's path crosses the recurrence forwards and backwards.
"""

import numpy as np
import torch

E = 2.0 ** -24


def half_step(dtype):
    """Largest relative error of one rounding to dtype (0 for float32: counted in k e)."""
    return torch.finfo(dtype).eps / 2 if dtype != torch.float32 else E


def norm(x, w, b, eps, rms, g=None):
    x, w = x.double(), w.double()
    mu = torch.zeros(x.shape[0], 1, dtype=torch.float64) if rms else x.mean(1, keepdim=True)
    r = ((x - mu).square().mean(1, keepdim=True) + eps) ** -0.5
    xh = (x - mu) * r
    y = xh * w + (0 if b is None else b.double())
    if g is None:
        return y
    g = g.double()
    q = g * w
    mq = torch.zeros_like(mu) if rms else q.mean(1, keepdim=True)
    dx = r * (q - mq - xh * (q * xh).mean(1, keepdim=True))
    return y, dx, (g * xh).sum(0), g.sum(0)


def _lens(lengths, B, L):
    return [L] * B if lengths is None else [min(max(int(v), 0), L) for v in lengths]


def conv(x, w, b, silu, state, lengths, g=None):
    """(y, state, dx, dw, db); gradients None without g."""
    x, w = x.double(), w.double()
    B, L, D = x.shape
    K = w.shape[1]
    b = torch.zeros(D, dtype=torch.float64) if b is None else b.double()
    past = torch.zeros(B, K - 1, D, dtype=torch.float64) if state is None else state.double()
    y, new = torch.zeros_like(x), past.clone()
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)
    for i, n in enumerate(_lens(lengths, B, L)):
        rows = torch.cat([past[i], x[i, :n]])
        new[i] = rows[n:n + K - 1]
        for t in range(n):
            win = rows[t:t + K]                                  # (K, D)
            p = b + (win * w.T).sum(0)
            s = 1 / (1 + torch.exp(-p))
            y[i, t] = p * s if silu else p
            if g is not None:
                q = g[i, t].double() * (s * (1 + p * (1 - s)) if silu else 1.0)
                db += q
                dw += (q * win).T
                for k in range(K):
                    at = t - (K - 1) + k
                    if at >= 0:
                        dx[i, at] += q * w[:, k]
    return (y, new, dx, dw, db) if g is not None else (y, new, None, None, None)


def softplus(x):
    return torch.where(x > 20, x, torch.log1p(torch.exp(x.clamp(max=20))))


def scan(u, dt, A, Bm, Cm, D=None, z=None, dt_bias=None, sp=True, state=None, lengths=None, g=None,
         magnitude=False):
    """Dict of y, h and, with g, du, ddt, dA, dB, dC, dD, dbias, dz.

    ``magnitude``: the sums of absolute values of the same formulas' paths."""
    m = torch.abs if magnitude else (lambda v: v)
    u, dt, A, Bm, Cm = (t.double() for t in (u, dt, A, Bm, Cm))
    B, L, d = u.shape
    N = A.shape[1]
    zero = torch.zeros(d, dtype=torch.float64)
    Dk = zero if D is None else D.double()
    raw = dt + (zero if dt_bias is None else dt_bias.double())
    de = softplus(raw) if sp else raw
    slope = torch.where(raw > 20, torch.ones_like(raw), torch.sigmoid(raw)) if sp \
        else torch.ones_like(raw)
    if z is not None:
        z = z.double()
        s = torch.sigmoid(z)
        gate, dgate = z * s, s * (1 + z * (1 - s))
    else:
        gate, dgate = torch.ones_like(u), torch.zeros_like(u)
    h = torch.zeros(B, d, N, dtype=torch.float64) if state is None else m(state.double())
    live = torch.tensor([[t < n for t in range(L)] for n in _lens(lengths, B, L)],
                        dtype=torch.bool).view(B, L, 1)
    uu, bb, cc, dk, dd, aa = m(u), m(Bm), m(Cm), m(Dk), m(de), m(A)
    gate_m, dgate_m = m(gate), dgate
    if magnitude and z is not None:   # s + s z (1 - s): its two paths cancel near z = -1.28
        dgate_m = s * (1 + z.abs() * (1 - s))
    before, after, yp = [], [], torch.zeros_like(u)
    for t in range(L):
        before.append(h)
        new = torch.exp(de[:, t, :, None] * A) * h + (dd[:, t] * uu[:, t])[..., None] \
            * bb[:, t, None, :]
        h = torch.where(live[:, t, :, None], new, h)
        after.append(h)
        yp[:, t] = torch.where(live[:, t], (h * cc[:, t, None, :]).sum(-1) + dk * uu[:, t], 0)
    out = {"y": yp * torch.where(live, gate_m, 0), "h": h}
    if g is None:
        return out
    g = torch.where(live, m(g.double()), 0)
    gy = g * gate_m
    q = torch.zeros_like(h)
    for k, t in dict(du=u, ddt=u, dB=Bm, dC=Cm).items():
        out[k] = torch.zeros_like(t)
    out["dA"] = torch.zeros_like(A)
    for t in range(L - 1, -1, -1):
        lt = live[:, t]
        gate_t = torch.exp(de[:, t, :, None] * A)
        q = q + gy[:, t, :, None] * cc[:, t, None, :]
        ql = q * lt[..., None]
        out["dC"][:, t] = (gy[:, t, :, None] * after[t]).sum(1)
        out["dB"][:, t] = (ql * (dd[:, t] * uu[:, t])[..., None]).sum(1)
        s1 = (ql * bb[:, t, None, :]).sum(-1)
        w = ql * gate_t * before[t]
        out["du"][:, t] = dk * gy[:, t] + dd[:, t] * s1
        out["ddt"][:, t] = (uu[:, t] * s1 + (w * aa).sum(-1)) * slope[:, t]
        out["dA"] += (w * dd[:, t, :, None]).sum(0)
        q = torch.where(lt[..., None], gate_t * q, q)
    out["ddt"] = torch.where(live, out["ddt"], 0)
    out["dD"] = (gy * torch.where(live, uu, 0)).sum((0, 1))
    out["dbias"] = out["ddt"].sum((0, 1))
    out["dz"] = g * yp * dgate_m
    return out


def token_step(h, u, dt, A, Bm, Cm, D=None, z=None, dt_bias=None, sp=True, magnitude=False):
    """(y, h) of one token: the scan over one step."""
    one = lambda t: None if t is None else t[:, None]  # noqa: E731
    r = scan(one(u), one(dt), A, one(Bm), one(Cm), D, one(z), dt_bias, sp, h, magnitude=magnitude)
    return r["y"][:, 0], r["h"]


def kept_weights(x, temperature, top_k, top_p, min_p):
    """The weights (0: not kept) of one row's tokens, float64; None without candidates."""
    x = np.array(x, dtype=np.float64)
    x[np.isnan(x)] = -np.inf
    V = len(x)
    if not (x > -np.inf).any():
        return None
    order = np.lexsort((np.arange(V), -x))
    order = order[x[order] > -np.inf]
    w = np.zeros(V)
    if not temperature > 0:
        w[order[0]] = 1.0
        return w
    top = x[order[0]]
    with np.errstate(invalid="ignore"):
        v = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / temperature))
    n = len(order) if top_k <= 0 else min(top_k, len(order))
    if top_p < 1:
        run, total = 0.0, v[:n].sum()
        for i in range(n):
            run += v[i]
            if run >= top_p * total:
                n = i + 1
                break
    for i in range(n):
        if v[i] >= min(min_p, 1.0):
            w[order[i]] = v[i]
    return w


def draw(w, u):
    """The token of the kept weights w at u, and how near u is to a border (relative)."""
    if w is None:
        return -1, 1.0
    cum = np.cumsum(w)
    over = np.nonzero((cum > u * cum[-1]) & (w > 0))[0]
    token = over[0] if len(over) else np.nonzero(w)[0][-1]
    return int(token), float(np.abs(cum[w > 0] / cum[-1] - u).min())
