"""Cases of the sequence-model operators: norms with their backward pass, the
short causal convolution and the selective scan (prompts, training, single
tokens), and drawing a token from a head's logits.

``run`` computes each operator in its plain form from elementary torch
operations in 32 bits (64 where a border decides), or, where ``own`` is true,
by the calls a user makes of this package.
"""

import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # one lockstep step of eight search lines: the pre-norm of a layer
        dict(name="norm_step", op="norm", kind="rms", rows=8, d=512, dtype="f32", grad=False),
        # a head's layer norm in training, odd sizes
        dict(name="norm_ragged", op="norm", kind="layer", rows=10007, d=1001, dtype="f32",
             grad=True),
        # the pre-norm of a layer in training, 2048 rows of 64 tokens
        dict(name="norm_train", op="norm", kind="rms", rows=131072, d=768, dtype="bf16", grad=True),
        # priming a ragged batch of prompts after an earlier part of each
        dict(name="conv_prompts", op="conv", B=37, L=333, D=1024, K=4, dtype="f32", ragged=True,
             state=True, grad=False),
        # a training micro-batch
        dict(name="conv_train", op="conv", B=512, L=64, D=1536, K=4, dtype="bf16", ragged=False,
             state=False, grad=True),
        # priming one long prompt
        dict(name="scan_prompt", op="scan", B=1, L=4096, D=1024, N=16, dtype="bf16", ragged=False,
             state=False, gate=True, grad=False),
        # training on many short rows
        dict(name="scan_train_rows", op="scan", B=256, L=64, D=1536, N=32, dtype="bf16",
             ragged=False, state=False, gate=True, grad=True),
        # training on a few long ones of odd lengths
        dict(name="scan_train_long", op="scan", B=2, L=4001, D=1536, N=16, dtype="f32",
             ragged=True, state=False, gate=True, grad=True),
        # one token of one line: the convolution's and the scan's step
        dict(name="token_one", op="token", B=1, D=1024, N=16, K=4, dtype="f32"),
        # one token of a large lockstep batch
        dict(name="token_batch", op="token", B=2048, D=1024, N=32, K=4, dtype="bf16"),
        # drawing the next move of eight lines
        dict(name="sample_few", op="sample", rows=8, V=8192, dtype="f32", temperature=0.8, top_k=50,
             top_p=0.9, min_p=0.0, per_row=False, masked=0.0),
        # drawing for a large batch of rollouts, each row with its own settings
        dict(name="sample_batch", op="sample", rows=4096, V=8192, dtype="bf16", temperature=1.0,
             top_k=0, top_p=0.95, min_p=0.02, per_row=True, masked=0.3),
    ]


def _spread(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "conv", "scan", "scan", "token", "sample"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "norm":
        d = _spread(rng, 64, 8192)
        return dict(op=op, kind=rng.choice(["rms", "layer"]), d=d,
                    rows=_spread(rng, 1, min(131072, 90_000_000 // d)), dtype=dtype,
                    grad=rng.random() < 0.6)
    if op == "conv":
        L, D = _spread(rng, 1, 4096), _spread(rng, 64, 4096)
        return dict(op=op, B=_spread(rng, 1, max(1, min(512, 48_000_000 // (L * D)))), L=L, D=D,
                    K=rng.randint(2, 4), dtype=dtype, ragged=rng.random() < 0.4,
                    state=rng.random() < 0.4, grad=rng.random() < 0.5)
    if op == "scan":
        L, D, N = _spread(rng, 1, 4096), _spread(rng, 64, 2048), rng.choice([8, 16, 16, 24, 32, 64])
        return dict(op=op, B=_spread(rng, 1, max(1, min(256, 400_000_000 // (L * D * N)))), L=L, D=D,
                    N=N, dtype=dtype, ragged=rng.random() < 0.4, state=rng.random() < 0.3,
                    gate=rng.random() < 0.7, grad=rng.random() < 0.5)
    if op == "token":
        D, N = _spread(rng, 64, 4096), rng.choice([8, 16, 16, 24, 32, 64])
        return dict(op=op, B=_spread(rng, 1, min(4096, 67_000_000 // (D * N))), D=D, N=N,
                    K=rng.randint(2, 4), dtype=dtype)
    V = _spread(rng, 32, 131072)
    return dict(op=op, rows=_spread(rng, 1, min(4096, 33_000_000 // V)), V=V, dtype=dtype,
                temperature=round(rng.uniform(0.3, 1.5), 3),
                top_k=rng.choice([0, 1, 20, 50, 1000]), top_p=rng.choice([1.0, 0.9, 0.5]),
                min_p=rng.choice([0.0, 0.0, 0.05]), per_row=rng.random() < 0.5,
                masked=rng.choice([0.0, 0.5, 0.99]))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0, dtype=torch.float32):
        return torch.randn(*shape, device="cuda", generator=g).mul_(scale).add_(shift).to(dtype)

    def uniform(*shape, lo=0.0, hi=1.0):
        return torch.rand(*shape, device="cuda", generator=g).mul_(hi - lo).add_(lo)

    s = dict(case)
    op = case["op"]
    if op == "norm":
        rows, d = case["rows"], case["d"]
        s["x"] = normal(rows, d, scale=1.5, shift=0.3, dtype=dt)
        s["w"] = normal(d, scale=0.2, shift=1.0)
        s["b"] = normal(d, scale=0.2) if case["kind"] == "layer" else None
        s["eps"] = 1e-5
        s["g"] = normal(rows, d, dtype=dt) if case["grad"] else None
        return s
    if op == "sample":
        rows, V = case["rows"], case["V"]
        logits = normal(rows, V, scale=2.5, dtype=dt)
        if case["masked"] > 0:   # moves that are not allowed
            logits.masked_fill_(uniform(rows, V) < case["masked"], float("-inf"))
        s["logits"] = logits
        s["u"] = uniform(rows)
        s["set"] = [case["temperature"], case["top_k"], case["top_p"], case["min_p"]]
        if case["per_row"]:
            s["set"] = [case["temperature"] * uniform(rows, lo=0.5, hi=1.5),
                        torch.randint(0, max(1, 2 * case["top_k"]) + 1, (rows,), device="cuda",
                                      generator=g, dtype=torch.int32),
                        case["top_p"] * uniform(rows, lo=0.8, hi=1.0),
                        case["min_p"] * uniform(rows, lo=0.5, hi=1.5)]
        return s
    B, D = case["B"], case["D"]
    if op in ("conv", "token"):
        K = case["K"]
        s["w"] = uniform(D, K, lo=-1.0, hi=1.0) / math.sqrt(K)
        s["b"] = uniform(D, lo=-0.5, hi=0.5)
    if op in ("scan", "token"):
        N = case["N"]
        # eigenvalues -1 .. -N, step sizes between 1e-3 and 1e-1
        s["A"] = -torch.arange(1, N + 1, device="cuda", dtype=torch.float32).repeat(D, 1) \
            * uniform(D, N, lo=0.8, hi=1.2)
        s["D"] = normal(D, scale=0.2, shift=1.0)
        d0 = torch.exp(uniform(D, lo=math.log(1e-3), hi=math.log(1e-1)))
        s["dt_bias"] = d0 + torch.log(-torch.expm1(-d0))
    if op == "token":
        s["conv_state"] = normal(B, K - 1, D, dtype=dt)
        s["x"] = normal(B, D, dtype=dt)
        s["h"] = normal(B, D, N, scale=0.3)
        # the halves of one projection's rows, and the columns of another's
        s["u"], s["z"] = normal(B, 2 * D, dtype=dt).split(D, dim=1)
        s["dt"] = normal(B, D, scale=0.5, dtype=dt)
        s["Bm"], s["Cm"] = normal(B, 2 * N, dtype=dt).split(N, dim=1)
        return s
    L = case["L"]
    s["lengths"] = None
    if case["ragged"]:
        s["lengths"] = torch.randint(0, L + 1, (B,), device="cuda", generator=g, dtype=torch.int32)
        s["lengths"][0] = L
    s["state"] = None
    if op == "conv":
        s["x"] = normal(B, L, 2 * D, dtype=dt)[..., :D]
        if case["state"]:
            s["state"] = normal(B, K - 1, D, dtype=dt)
    else:
        s["u"] = normal(B, L, D, dtype=dt)
        s["z"] = normal(B, L, 2 * D, dtype=dt)[..., D:] if case["gate"] else None
        s["dt"] = normal(B, L, D, scale=0.5, dtype=dt)
        s["Bm"], s["Cm"] = normal(B, L, 2 * N, dtype=dt).split(N, dim=2)
        if case["state"]:
            s["state"] = normal(B, D, N, scale=0.3)
    s["g"] = normal(B, L, D, dtype=dt) if case["grad"] else None
    if case["grad"]:   # a training program's leaves
        for k in ("x", "u", "dt", "z", "Bm", "Cm", "w", "b", "A", "D", "dt_bias"):
            if torch.is_tensor(s.get(k)):
                s[k].requires_grad_(True)
    return s


# ---------------------------------------------------------------- plain forms

def _norm_plain(s):
    x, w, b = s["x"].float(), s["w"], s["b"]
    dt = s["x"].dtype
    layer = s["kind"] == "layer"
    xc = x - x.mean(-1, keepdim=True) if layer else x
    r = torch.rsqrt(xc.square().mean(-1, keepdim=True) + s["eps"])
    xh = xc * r
    y = xh * w + b if layer else xh * w
    if s["g"] is None:
        return {"y": y.to(dt)}
    g = s["g"].float()
    gw = g * w
    dx = gw - xh * (gw * xh).mean(-1, keepdim=True)
    if layer:
        dx = dx - gw.mean(-1, keepdim=True)
    out = {"y": y.to(dt), "dx": (dx * r).to(dt), "dw": (g * xh).sum(0)}
    if layer:
        out["db"] = g.sum(0)
    return out


def _silu(x):
    return x * torch.sigmoid(x)


def _dsilu(x):
    sg = torch.sigmoid(x)
    return sg * (1 + x * (1 - sg))


def _softplus(x):
    return torch.where(x > 20, x, torch.log1p(torch.exp(torch.clamp(x, max=20.0))))


def _valid(s, L):
    """(B, L, 1): the steps before each row's length."""
    if s["lengths"] is None:
        return None
    return (torch.arange(L, device="cuda") < s["lengths"][:, None])[..., None]


def _conv_plain(s):
    x, w, b = s["x"].detach(), s["w"].detach(), s["b"].detach()
    dt, (B, L, D), K = x.dtype, x.shape, w.shape[1]
    head = s["state"] if s["state"] is not None else x.new_zeros(B, K - 1, D)
    rows = torch.cat([head, x], 1)
    win = rows.float().unfold(1, K, 1)                       # (B, L, D, K)
    p = (win * w).sum(-1) + b
    ok = _valid(s, L)
    y = _silu(p) if ok is None else torch.where(ok, _silu(p), torch.zeros_like(p))
    if s["g"] is None:
        n = s["lengths"].long() if ok is not None else torch.full((B,), L, device="cuda")
        at = n[:, None] + torch.arange(K - 1, device="cuda")
        return {"y": y.to(dt), "state": rows.gather(1, at[..., None].expand(B, K - 1, D))}
    g = s["g"].float() * _dsilu(p)
    if ok is not None:
        g = g * ok
    after = torch.cat([g, g.new_zeros(B, K - 1, D)], 1).unfold(1, K, 1)
    return {"y": y.to(dt), "dx": (after * w.flip(1)).sum(-1).to(dt),
            "dw": (g[..., None] * win).sum((0, 1)), "db": g.sum((0, 1))}


def _recurrence(a, b):
    """h[t] = a[t] h[t-1] + b[t] along dim 1, by doubling; h[-1] = 0."""
    L, step = a.shape[1], 1
    while step < L:
        b = torch.cat([b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]], 1)
        if 2 * step < L:
            a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return b


def _scan_plain(s):
    det = {k: s[k].detach().float() for k in ("u", "dt", "Bm", "Cm")}
    u, Bm, Cm = det["u"], det["Bm"], det["Cm"]
    A, Dk, bias = s["A"].detach(), s["D"].detach(), s["dt_bias"].detach()
    z = s["z"].detach().float() if s["z"] is not None else None
    dt, (B, L, D) = s["u"].dtype, u.shape
    raw = det["dt"] + bias
    de = _softplus(raw)
    ok = _valid(s, L)
    if ok is not None:   # a step of size zero leaves the state as it is
        de = de * ok
    a = torch.exp(de[..., None] * A)
    b = (de * u)[..., None] * Bm[:, :, None, :]
    if s["state"] is not None:
        b[:, 0] += a[:, 0] * s["state"]
    h = _recurrence(a, b)
    del b
    yp = (h * Cm[:, :, None, :]).sum(-1) + Dk * u
    y = yp * _silu(z) if z is not None else yp
    if ok is not None:
        y = y * ok
    if s["g"] is None:
        return {"y": y.to(dt), "state": h[:, -1].clone()}
    g = s["g"].float()
    if ok is not None:
        g = g * ok
    gy = g * _silu(z) if z is not None else g
    # the state's gradient runs the same recurrence from the back
    back = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1).flip(1)
    dh = _recurrence(back, (gy[..., None] * Cm[:, :, None, :]).flip(1)).flip(1)
    del back
    out = {"y": y.to(dt)}
    dC = (h * gy[..., None]).sum(2)
    head = s["state"] if s["state"] is not None else torch.zeros_like(h[:, 0])
    ha = torch.cat([head[:, None], h[:, :-1]], 1).mul_(a).mul_(dh)  # dh h[t-1] a
    del h, a
    dB = (dh * (de * u)[..., None]).sum(2)
    dhB = (dh * Bm[:, :, None, :]).sum(-1)
    del dh
    dA = (ha * de[..., None]).sum((0, 1))
    dde = u * dhB + (ha * A).sum(-1)
    draw_ = dde * torch.where(raw > 20, torch.ones_like(raw), torch.sigmoid(raw))
    if ok is not None:
        draw_, dB = draw_ * ok, dB * ok
    out.update(du=(Dk * gy + de * dhB).to(dt), ddt=draw_.to(dt), dA=dA, dB=dB.to(dt), dC=dC.to(dt),
               dD=(gy * u).sum((0, 1)), dbias=draw_.sum((0, 1)))
    if z is not None:
        out["dz"] = (g * yp * _dsilu(z)).to(dt)
    return out


def _token_plain(s):
    x, dt = s["x"].float(), s["x"].dtype
    rows = torch.cat([s["conv_state"], s["x"][:, None]], 1)
    c = _silu((rows.float().transpose(1, 2) * s["w"]).sum(-1) + s["b"]).to(dt)
    s["conv_state"].copy_(rows[:, 1:])
    u, z = s["u"].float(), s["z"].float()
    de = _softplus(s["dt"].float() + s["dt_bias"])
    a = torch.exp(de[..., None] * s["A"])
    h = a * s["h"] + (de * u)[..., None] * s["Bm"].float()[:, None, :]
    s["h"].copy_(h)
    y = ((h * s["Cm"].float()[:, None, :]).sum(-1) + s["D"] * u) * _silu(z)
    return {"conv": c, "conv_state": s["conv_state"], "y": y.to(dt), "h": s["h"]}


def _sample_plain(s):
    x = s["logits"].double()
    rows, V = x.shape
    T, k, p, mp = (v.double()[:, None] if torch.is_tensor(v)
                   else torch.full((rows, 1), float(v), dtype=torch.float64, device="cuda")
                   for v in s["set"])
    x = torch.where(torch.isnan(x), torch.full_like(x, float("-inf")), x)
    top = x.max(1, keepdim=True).values
    xs, order = torch.sort(x, dim=1, descending=True, stable=True)
    ws = torch.where(xs == top, torch.ones_like(xs), torch.exp((xs - top) / T))
    place = torch.arange(V, device="cuda")
    keep = (xs > float("-inf")) & ((k <= 0) | (place < k))
    ws = ws * keep
    total = ws.cumsum(1)
    before = torch.cat([torch.zeros_like(total[:, :1]), total[:, :-1]], 1)
    keep &= (place == 0) | (p >= 1) | (before < p * total[:, -1:])
    keep &= ws >= mp.clamp(max=1.0)
    w = torch.zeros_like(ws).scatter_(1, order, ws * keep)
    cum = w.cumsum(1)
    over = (cum > s["u"].double()[:, None] * cum[:, -1:]) & (w > 0)
    token = torch.where(over.any(1), over.int().argmax(1), V - 1 - (w > 0).int().flip(1).argmax(1))
    return {"token": torch.where((w > 0).any(1), token, torch.full_like(token, -1))}


# ---------------------------------------------------------------- the package's calls

def _own(s):
    op = s["op"]
    if op == "norm":
        from redpanda_b200.norm import m3_layer_norm, m3_rms_norm
        if s["g"] is None:
            if s["kind"] == "layer":
                return {"y": m3_layer_norm(s["x"], s["w"], s["b"], eps=s["eps"])}
            return {"y": m3_rms_norm(s["x"], s["w"], eps=s["eps"])}
        x, w = s["x"].detach().requires_grad_(True), s["w"].detach().requires_grad_(True)
        if s["kind"] == "layer":
            b = s["b"].detach().requires_grad_(True)
            y = m3_layer_norm(x, w, b, eps=s["eps"])
            dx, dw, db = torch.autograd.grad(y, (x, w, b), s["g"])
            return {"y": y, "dx": dx, "dw": dw, "db": db}
        y = m3_rms_norm(x, w, eps=s["eps"])
        dx, dw = torch.autograd.grad(y, (x, w), s["g"])
        return {"y": y, "dx": dx, "dw": dw}
    if op == "sample":
        from redpanda_b200.sampling import m3_sample
        T, k, p, mp = s["set"]
        return {"token": m3_sample(s["logits"], s["u"], temperature=T, top_k=k, top_p=p, min_p=mp)}
    from redpanda_b200 import selective as S
    if op == "token":
        c = S.m3_causal_conv_step_(s["conv_state"], s["x"], s["w"], s["b"])
        y = S.m3_selective_step_(s["h"], s["u"], s["dt"], s["A"], s["Bm"], s["Cm"], D=s["D"],
                                 z=s["z"], dt_bias=s["dt_bias"])
        return {"conv": c, "conv_state": s["conv_state"], "y": y, "h": s["h"]}
    if op == "conv":
        if s["g"] is None:
            y, state = S.m3_causal_conv_with_state(s["x"], s["w"], s["b"], state=s["state"],
                                                   lengths=s["lengths"])
            return {"y": y, "state": state}
        y = S.m3_causal_conv(s["x"], s["w"], s["b"], state=s["state"], lengths=s["lengths"])
        dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["g"])
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    kw = dict(D=s["D"], z=s["z"], dt_bias=s["dt_bias"], state=s["state"], lengths=s["lengths"])
    args = (s["u"], s["dt"], s["A"], s["Bm"], s["Cm"])
    if s["g"] is None:
        y, state = S.m3_selective_scan_with_state(*args, **kw)
        return {"y": y, "state": state}
    y = S.m3_selective_scan(*args, **kw)
    leaves = dict(du=s["u"], ddt=s["dt"], dA=s["A"], dB=s["Bm"], dC=s["Cm"], dD=s["D"],
                  dbias=s["dt_bias"])
    if s["z"] is not None:
        leaves["dz"] = s["z"]
    grads = torch.autograd.grad(y, list(leaves.values()), s["g"])
    return {"y": y, **dict(zip(leaves, grads))}


_PLAIN = {"norm": _norm_plain, "conv": _conv_plain, "scan": _scan_plain, "token": _token_plain,
          "sample": _sample_plain}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _PLAIN[state["op"]](state)


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    op = case["op"]
    if op == "norm":
        n = case["rows"] * case["d"]
        return {"bytes": n * e * (5 if case["grad"] else 2) + 8 * case["d"],
                "flops": n * (20 if case["grad"] else 7)}
    if op == "sample":
        return {"bytes": case["rows"] * (case["V"] * e + 24), "flops": 4 * case["rows"] * case["V"]}
    B, D = case["B"], case["D"]
    if op == "token":
        K, N = case["K"], case["N"]
        return {"bytes": B * D * (e * (2 * K + 4) + 8 * N) + B * N * 2 * e + D * (4 * N + 4 * K + 12),
                "flops": B * D * (7 * N + 2 * K + 20)}
    n = B * case["L"] * D
    if op == "conv":
        K = case["K"]
        return {"bytes": n * e * (5 if case["grad"] else 2) + D * 4 * (K + 1),
                "flops": n * (6 * K + 20 if case["grad"] else 2 * K + 5)}
    N, arrays = case["N"], 3 + case["gate"]
    rows = B * case["L"] * N * 2 * e
    if case["grad"]:   # forward: u, dt, z in, y out; backward: these and dy in, their gradients out
        return {"bytes": n * e * (2 * arrays + 2 + case["gate"]) + 3 * rows + 8 * D * N,
                "flops": n * (25 * N + 40)}
    return {"bytes": n * e * arrays + rows + 4 * D * N * (1 + B), "flops": n * (7 * N + 15)}


# ---------------------------------------------------------------- from the definitions, in 64 bits

def exact(case, seed):
    """Steps one at a time in 64 bits; None for drawn tokens (whole numbers)."""
    op = case["op"]
    if op == "sample":
        return None
    s = prepare(case, seed)
    d = {k: (v.detach().double() if torch.is_tensor(v) and v.is_floating_point() else v)
         for k, v in s.items()}
    with torch.no_grad():
        return {"norm": _norm_exact, "conv": _conv_exact, "scan": _scan_exact,
                "token": _token_exact}[op](d)


def _norm_exact(d):
    x, w, n = d["x"], d["w"], d["x"].shape[1]
    mu = x.sum(1) / n if d["kind"] == "layer" else torch.zeros_like(x[:, 0])
    sd = (((x - mu[:, None]) ** 2).sum(1) / n + d["eps"]).sqrt()
    xh = (x - mu[:, None]) / sd[:, None]
    out = {"y": xh * w + (d["b"] if d["kind"] == "layer" else 0.0)}
    if d["g"] is None:
        return out
    q = d["g"] * w
    along = torch.einsum("rd,rd->r", q, xh) / n
    mean = q.sum(1) / n if d["kind"] == "layer" else torch.zeros_like(along)
    out["dx"] = (q - mean[:, None] - xh * along[:, None]) / sd[:, None]
    out["dw"] = torch.einsum("rd,rd->d", d["g"], xh)
    if d["kind"] == "layer":
        out["db"] = torch.einsum("rd->d", d["g"])
    return out


def _conv_exact(d):
    x, w, b = d["x"], d["w"], d["b"]
    (B, L, D), K = x.shape, w.shape[1]
    n = (d["lengths"].tolist() if d["lengths"] is not None else [L] * B)
    past = d["state"] if d["state"] is not None else x.new_zeros(B, K - 1, D)
    y = torch.zeros_like(x)
    grad = d["g"] is not None
    state, dx, dw, db = past.clone(), torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)
    for i in range(B):
        m = n[i]
        rows = torch.cat([past[i], x[i, :m]])
        state[i] = rows[m:m + K - 1]
        if m == 0:
            continue
        p = b.expand(m, D).clone()
        for k in range(K):
            p += rows[k:k + m] * w[:, k]
        sg = 1 / (1 + (-p).exp())
        y[i, :m] = p * sg
        if grad:
            q = d["g"][i, :m] * (sg + p * sg * (1 - sg))
            db += q.sum(0)
            for k in range(K):
                dw[:, k] += (q * rows[k:k + m]).sum(0)
                lag = K - 1 - k
                if m > lag:
                    dx[i, :m - lag] += q[lag:] * w[:, k]
    return {"y": y, "dx": dx, "dw": dw, "db": db} if grad else {"y": y, "state": state}


def _scan_exact(d):
    u, A, Bm, Cm, g = d["u"], d["A"], d["Bm"], d["Cm"], d["g"]
    (B, L, D), N = u.shape, A.shape[1]
    raw = d["dt"] + d["dt_bias"]
    de = torch.nn.functional.softplus(raw, threshold=40)
    n = d["lengths"] if d["lengths"] is not None else torch.full((B,), L, device="cuda")
    z = d["z"]
    sg = 1 / (1 + (-z).exp()) if z is not None else None
    h = d["state"].clone() if d["state"] is not None else u.new_zeros(B, D, N)
    grad = g is not None
    yp = torch.zeros_like(u)
    kept = torch.zeros(L, B, D, N, dtype=torch.float64, device="cuda") if grad else None
    for t in range(L):
        live = (t < n)[:, None]
        if grad:
            kept[t] = h
        new = (de[:, t, :, None] * A).exp() * h \
            + (de[:, t] * u[:, t])[..., None] * Bm[:, t, None, :]
        h = torch.where(live[..., None], new, h)
        yp[:, t] = torch.where(live, torch.einsum("bdn,bn->bd", h, Cm[:, t]) + d["D"] * u[:, t], 0)
    y = yp * z * sg if z is not None else yp
    if not grad:
        return {"y": y, "state": h}
    out = {"y": y, "du": torch.zeros_like(u), "ddt": torch.zeros_like(u), "dA": torch.zeros_like(A),
           "dB": torch.zeros_like(Bm), "dC": torch.zeros_like(Cm), "dD": torch.zeros_like(d["D"]),
           "dbias": torch.zeros_like(d["D"])}
    if z is not None:
        out["dz"] = g * yp * (sg + z * sg * (1 - sg))
    q = torch.zeros_like(h)
    for t in range(L - 1, -1, -1):
        live = (t < n)[:, None]
        gt = torch.where(live, g[:, t] * (z[:, t] * sg[:, t] if z is not None else 1.0), 0)
        a = (de[:, t, :, None] * A).exp()
        now = a * kept[t] + (de[:, t] * u[:, t])[..., None] * Bm[:, t, None, :]
        q = q + gt[..., None] * Cm[:, t, None, :]
        out["dC"][:, t] = torch.einsum("bd,bdn->bn", gt, now) * live
        ql = q * live[..., None]
        through = torch.einsum("bdn,bn->bd", ql, Bm[:, t])
        out["dB"][:, t] = torch.einsum("bdn,bd->bn", ql, de[:, t] * u[:, t])
        qa = ql * kept[t] * a
        out["dA"] += torch.einsum("bdn,bd->dn", qa, de[:, t])
        out["du"][:, t] = d["D"] * gt + de[:, t] * through
        r = (u[:, t] * through + torch.einsum("bdn,dn->bd", qa, A)) / (1 + (-raw[:, t]).exp())
        out["ddt"][:, t] = r
        out["dbias"] += r.sum(0)
        out["dD"] += (gt * u[:, t]).sum(0)
        q = torch.where(live[..., None], a * q, q)
    return out


def _token_exact(d):
    rows = torch.cat([d["conv_state"], d["x"][:, None]], 1)
    p = torch.einsum("bkd,dk->bd", rows, d["w"]) + d["b"]
    de = torch.nn.functional.softplus(d["dt"] + d["dt_bias"], threshold=40)
    h = torch.exp(torch.einsum("bd,dn->bdn", de, d["A"])) * d["h"] \
        + torch.einsum("bd,bd,bn->bdn", de, d["u"], d["Bm"])
    y = torch.einsum("bdn,bn->bd", h, d["Cm"]) + d["D"] * d["u"]
    return {"conv": p / (1 + (-p).exp()), "conv_state": rows[:, 1:],
            "y": y * d["z"] / (1 + (-d["z"]).exp()), "h": h}
