"""Cases of the operators of a gated recurrent layer: the RMS norm with the
residual's addition (and its backward pass, and its result in 8 bits with
scales), the gated linear recurrence (prompts, training, single tokens) and the
product of a few rows with 4-bit weights and group scales.

``run`` computes each operator in its plain form from elementary torch
operations in 32 bits, or, where ``own`` is true, by the calls a user makes of
this package.
"""

import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # one lockstep step of eight search lines: residual and pre-norm of a layer
        dict(name="addnorm_step", op="addnorm", rows=8, d=512, x="f32", stream="f32", y="f32",
             grad=False),
        # training at odd sizes in 32 bits
        dict(name="addnorm_ragged", op="addnorm", rows=10007, d=1001, x="f32", stream="f32",
             y="f32", grad=True),
        # training under autocast: 2048 rows of 64 tokens, a bf16 branch into an fp32 stream
        dict(name="addnorm_train", op="addnorm", rows=131072, d=768, x="bf16", stream="f32",
             y="bf16", grad=True),
        # a few lines' input rows for an 8-bit projection, a scale per row
        dict(name="norm8_step", op="norm8", rows=8, d=768, x="f32", stream="", group=0),
        # the same for a batch of prompts, with the residual and a scale per 128 columns
        dict(name="norm8_prompts", op="norm8", rows=16384, d=4096, x="bf16", stream="bf16",
             group=128),
        # priming one long prompt
        dict(name="gated_prompt", op="gated", B=1, L=16384, D=1024, dtype="bf16", ragged=False,
             state=False, grad=False),
        # training on many short rows
        dict(name="gated_train_rows", op="gated", B=256, L=64, D=2048, dtype="bf16", ragged=False,
             state=False, grad=True),
        # training on a few long ones of odd lengths
        dict(name="gated_train_long", op="gated", B=2, L=16001, D=1280, dtype="f32", ragged=True,
             state=False, grad=True),
        # one token of a large lockstep batch
        dict(name="gated_token", op="token", B=2048, D=2048, dtype="bf16"),
        # a search node's in_proj with the norm ahead and silu behind
        dict(name="q4_node", op="q4", rows=1, K=384, N=1536, group=64, dtype="f32", norm=True,
             split=True, center=True),
        # eight lines' logits over the moves
        dict(name="q4_lines", op="q4", rows=8, K=768, N=8192, group=64, dtype="f32", norm=False,
             split=False, center=True),
        # a large head for three rows
        dict(name="q4_large", op="q4", rows=3, K=8192, N=65536, group=128, dtype="bf16", norm=False,
             split=False, center=False),
    ]


def _spread(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["addnorm", "addnorm", "norm8", "gated", "gated", "gated", "token", "q4", "q4"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "addnorm":
        d = _spread(rng, 64, 8192)
        return dict(op=op, d=d, rows=_spread(rng, 1, min(131072, 80_000_000 // d)), x=dtype,
                    stream=rng.choice(["f32", "bf16"]), y=rng.choice(["f32", "bf16"]),
                    grad=rng.random() < 0.6)
    if op == "norm8":
        group = rng.choice([0, 0, 32, 64, 128])
        d = _spread(rng, 64, 8192) if not group else group * _spread(rng, 1, 8192 // group)
        return dict(op=op, d=d, rows=_spread(rng, 1, min(65536, 64_000_000 // d)), x=dtype,
                    stream=rng.choice(["", "f32", "bf16"]), group=group)
    if op == "gated":
        L = _spread(rng, 1, 65536)
        D = _spread(rng, 64, min(4096, 80_000_000 // L))
        return dict(op=op, L=L, D=D, B=_spread(rng, 1, max(1, min(512, 40_000_000 // (L * D)))),
                    dtype=dtype, ragged=rng.random() < 0.4, state=rng.random() < 0.4,
                    grad=L * D <= 40_000_000 and rng.random() < 0.5)
    if op == "token":
        D = _spread(rng, 64, 8192)
        return dict(op=op, D=D, B=_spread(rng, 1, min(4096, 8_000_000 // D)), dtype=dtype)
    K = _spread(rng, 32, 8192)
    N = _spread(rng, 16, min(65536, 400_000_000 // K))
    return dict(op=op, rows=rng.randint(1, 8), K=K, N=N, group=rng.choice([32, 64, 128]),
                dtype=dtype, norm=rng.random() < 0.5, split=rng.random() < 0.3,
                center=rng.random() < 0.6)


def _quantized(w, group, center):
    """4-bit codes of w (N, K), two to a byte (the first in the low half), and the
    scale and center of each group of columns: w ~ scale (code - 8) + center."""
    N, K = w.shape
    n = -(-K // group)
    pad = torch.nn.functional.pad(w, (0, n * group - K)).view(N, n, group)
    lo, hi = pad.amin(2), pad.amax(2)
    scale = ((hi - lo) / 15 if center else torch.maximum(hi / 7, -lo / 8)).clamp(min=1e-8)
    scale = scale.bfloat16()
    mid = (lo + 8 * scale.float() if center else torch.zeros_like(lo)).bfloat16()
    q = torch.round((pad - mid.float()[..., None]) / scale.float()[..., None]).add_(8).clamp_(0, 15)
    q = q.to(torch.uint8).view(N, n * group)[:, :K]
    q = torch.nn.functional.pad(q, (0, K & 1))
    return q[:, 0::2] | (q[:, 1::2] << 4), scale, (mid if center else None)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0, shift=0.0, dtype=torch.float32):
        return torch.randn(*shape, device="cuda", generator=g).mul_(scale).add_(shift).to(dtype)

    def uniform(*shape, lo=0.0, hi=1.0):
        return torch.rand(*shape, device="cuda", generator=g).mul_(hi - lo).add_(lo)

    s = dict(case)
    op = case["op"]
    if op in ("addnorm", "norm8"):
        rows, d = case["rows"], case["d"]
        s["branch"] = normal(rows, d, scale=0.5, dtype=_TYPES[case["x"]])
        s["res"] = None
        if case["stream"]:
            s["res"] = normal(rows, d, scale=1.5, shift=0.2, dtype=_TYPES[case["stream"]])
        s["w"] = normal(d, scale=0.2, shift=1.0)
        s["eps"] = 1e-5
        if case.get("grad"):
            s["gy"] = normal(rows, d, dtype=_TYPES[case["y"]])
            s["gs"] = normal(rows, d, dtype=_TYPES[case["stream"]])
            for k in ("branch", "res", "w"):   # a training program's leaves
                s[k].requires_grad_(True)
        return s
    dt = _TYPES[case["dtype"]]
    if op == "q4":
        rows, K, N = case["rows"], case["K"], case["N"]
        s["x"] = normal(rows, K, dtype=dt)
        packed, scale, center = _quantized(normal(N, K, scale=K ** -0.5), case["group"],
                                           case["center"])
        s["packed"], s["scale"], s["mid"] = packed, scale, center
        if own:   # the weights as the package lays them out, once
            from redpanda_b200.quant import Q4Weight
            s["weight"] = Q4Weight.from_packed(packed, scale, center, d_in=K, group=case["group"])
        s["bias"] = normal(N, scale=0.1)
        s["norm_w"] = normal(K, scale=0.2, shift=1.0) if case["norm"] else None
        s["eps"] = 1e-5
        s["cut"] = N // 2 if case["split"] else N
        return s
    B, D = case["B"], case["D"]
    # decays between about 0.9 and 0.999 per step with an open gate
    d0 = -torch.log(uniform(D, lo=0.9, hi=0.999)) / 8.0
    s["decay"] = torch.log(torch.expm1(d0))
    if op == "token":
        s["x"] = normal(B, D, dtype=dt)
        s["rg"], s["ig"] = normal(B, 2 * D, dtype=dt).split(D, dim=1)
        s["h"] = normal(B, D, scale=0.5)
        return s
    L = case["L"]
    s["x"] = normal(B, L, D, dtype=dt)
    s["rg"], s["ig"] = normal(B, L, 2 * D, dtype=dt).split(D, dim=2)
    s["state"] = normal(B, D, scale=0.5) if case["state"] else None
    s["lengths"] = None
    if case["ragged"]:
        s["lengths"] = torch.randint(0, L + 1, (B,), device="cuda", generator=g, dtype=torch.int32)
        s["lengths"][0] = L
    s["g"] = normal(B, L, D, dtype=dt) if case["grad"] else None
    if case["grad"]:
        for k in ("x", "rg", "ig", "decay"):
            s[k].requires_grad_(True)
    return s


# ---------------------------------------------------------------- plain forms

def _addnorm_plain(s):
    x, w = s["branch"].detach(), s["w"].detach()
    t = s["res"].dtype
    keep = (x.float() + s["res"].detach().float()).to(t)
    v = keep.float()
    r = torch.rsqrt(v.square().mean(-1, keepdim=True) + s["eps"])
    sh = v * r
    out = {"y": (sh * w).to(_TYPES[s["y"]]), "s": keep}
    if s["grad"]:
        gy = s["gy"].float()
        q = gy * w
        ds = s["gs"].float() + r * (q - sh * (q * sh).mean(-1, keepdim=True))
        out.update(dx=ds.to(x.dtype), dres=ds.to(t), dw=(gy * sh).sum(0))
    return out


def _norm8_plain(s):
    x, w, group = s["branch"], s["w"], s["group"]
    out = {}
    if s["res"] is not None:
        x = out["s"] = (x.float() + s["res"].float()).to(s["res"].dtype)
    v = x.float()
    y = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + s["eps"]) * w
    parts = y.view(y.shape[0], -1, group or y.shape[1])
    scale = (parts.abs().amax(-1) / 448.0).clamp(min=2.0 ** -126)
    out["q"] = (parts / scale[..., None]).view_as(y).to(torch.float8_e4m3fn)
    out["scale"] = scale
    return out


def _sigmoid(x):
    return 1 / (1 + torch.exp(-x))


def _softplus(x):
    return torch.where(x > 20, x, torch.log1p(torch.exp(torch.clamp(x, max=20.0))))


def _recurrence(a, b):
    """h[t] = a[t] h[t-1] + b[t] along dim 1, by doubling; h[-1] = 0."""
    L, step = a.shape[1], 1
    while step < L:
        b = torch.cat([b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]], 1)
        if 2 * step < L:
            a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return b


def _gates(s):
    x, rg, ig = (s[k].detach().float() for k in ("x", "rg", "ig"))
    r, i = _sigmoid(rg), _sigmoid(ig)
    k = -8.0 * _softplus(s["decay"].detach())
    return x, r, i, k * r


def _gated_plain(s):
    x, r, i, l = _gates(s)
    dt, (B, L, D) = s["x"].dtype, x.shape
    ok = None
    if s["lengths"] is not None:   # steps past a length leave the state as it is
        ok = (torch.arange(L, device="cuda") < s["lengths"][:, None])[..., None]
        l = l * ok
    a, m = torch.exp(l), torch.sqrt(-torch.expm1(2 * l))
    b = m * i * x
    if s["state"] is not None:
        b[:, 0] += a[:, 0] * s["state"]
    h = _recurrence(a, b)
    y = h if ok is None else h * ok
    if s["g"] is None:
        return {"y": y.to(dt), "state": h[:, -1].clone()}
    g = s["g"].float() if ok is None else s["g"].float() * ok
    back = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1).flip(1)
    q = _recurrence(back, g.flip(1)).flip(1)
    head = s["state"] if s["state"] is not None else torch.zeros_like(h[:, 0])
    before = torch.cat([head[:, None], h[:, :-1]], 1)
    inv = torch.where(m > 0, 1 / m, torch.zeros_like(m))
    e = q * l * (a * before - a * a * inv * i * x)
    d0 = s["decay"].detach()
    dec = (_sigmoid(d0) / _softplus(d0)) * e.sum((0, 1))
    qm = q * m
    return {"y": y.to(dt), "dx": (qm * i).to(dt), "drg": (e * (1 - r)).to(dt),
            "dig": (qm * x * i * (1 - i)).to(dt), "ddecay": dec}


def _token_plain(s):
    x, r, i, l = _gates(s)
    h = torch.exp(l) * s["h"] + torch.sqrt(-torch.expm1(2 * l)) * i * x
    s["h"].copy_(h)
    return {"y": h.to(s["x"].dtype), "h": s["h"]}


def _q4_plain(s):
    N, K, group = s["N"], s["K"], s["group"]
    p = s["packed"]
    q = torch.stack([p & 15, p >> 4], 2).view(N, -1)[:, :K].float() - 8
    n = s["scale"].shape[1]
    q = torch.nn.functional.pad(q, (0, n * group - K)).view(N, n, group)
    w = q * s["scale"].float()[..., None]
    if s["mid"] is not None:
        w += s["mid"].float()[..., None]
    w = w.view(N, n * group)[:, :K]
    x = s["x"].float()
    if s["norm_w"] is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + s["eps"]) * s["norm_w"]
    y = x @ w.t() + s["bias"]
    if not s["split"]:
        return {"y": y.to(s["x"].dtype)}
    u, z = y[:, :s["cut"]], y[:, s["cut"]:]
    return {"u": (u * _sigmoid(u)).to(s["x"].dtype), "z": z.to(s["x"].dtype)}


# ---------------------------------------------------------------- the package's calls

def _own(s):
    op = s["op"]
    if op == "addnorm":
        from redpanda_b200.norm import m3_add_rms_norm
        y, keep = m3_add_rms_norm(s["branch"], s["res"], s["w"], eps=s["eps"],
                                  out_dtype=_TYPES[s["y"]])
        out = {"y": y, "s": keep}
        if s["grad"]:
            out["dx"], out["dres"], out["dw"] = torch.autograd.grad(
                (y, keep), (s["branch"], s["res"], s["w"]), (s["gy"], s["gs"]))
        return out
    if op == "norm8":
        from redpanda_b200.norm import m3_rms_norm_8bit
        got = m3_rms_norm_8bit(s["branch"], s["w"], residual=s["res"], eps=s["eps"],
                               dtype=torch.float8_e4m3fn, group=s["group"] or None)
        return dict(zip(("q", "scale", "s"), got))
    if op == "q4":
        from redpanda_b200.quant import m3_rows_linear_q4
        u, z = m3_rows_linear_q4(s["x"], s["weight"], s["bias"], norm_weight=s["norm_w"],
                                 eps=s["eps"], split=s["cut"], silu=s["split"])
        return {"u": u, "z": z} if s["split"] else {"y": u}
    from redpanda_b200 import gated as G
    if op == "token":
        y = G.m3_gated_step_(s["h"], s["x"], s["rg"], s["ig"], s["decay"], c=8.0)
        return {"y": y, "h": s["h"]}
    args = (s["x"], s["rg"], s["ig"], s["decay"])
    kw = dict(c=8.0, state=s["state"], lengths=s["lengths"])
    if s["g"] is None:
        y, state = G.m3_gated_scan_with_state(*args, **kw)
        return {"y": y, "state": state}
    y = G.m3_gated_scan(*args, **kw)
    return {"y": y, **dict(zip(("dx", "drg", "dig", "ddecay"),
                               torch.autograd.grad(y, args, s["g"])))}


_PLAIN = {"addnorm": _addnorm_plain, "norm8": _norm8_plain, "gated": _gated_plain,
          "token": _token_plain, "q4": _q4_plain}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _PLAIN[state["op"]](state)


def _size(t):
    return {"f32": 4, "bf16": 2, "": 0}[t]


def work(case):
    op = case["op"]
    if op in ("addnorm", "norm8"):
        n = case["rows"] * case["d"]
        ex, es = _size(case["x"]), _size(case["stream"])
        if op == "norm8":   # x and the residual in, their sum, the codes and the scales out
            groups = case["rows"] * (case["d"] // case["group"] if case["group"] else 1)
            return {"bytes": n * (ex + 2 * es + 1) + 4 * groups + 4 * case["d"], "flops": 8 * n}
        ey = _size(case["y"])
        b, f = ex + 2 * es + ey, 6
        if case["grad"]:   # the sum and both gradients in, their sum out once per type
            b, f = b + 2 * es + ey + (es if ex == es else ex + es), f + 14
        return {"bytes": n * b + 8 * case["d"], "flops": f * n}
    e = _size(case["dtype"])
    if op == "q4":
        N, K = case["N"], case["K"]
        groups = N * -(-K // case["group"])
        return {"bytes": N * K // 2 + groups * (4 if case["center"] else 2)
                + case["rows"] * (N + K) * e + 4 * N, "flops": 2 * case["rows"] * N * K}
    n = case["B"] * case["D"]
    if op == "token":
        return {"bytes": n * (4 * e + 8), "flops": 30 * n}
    n *= case["L"]
    if case["grad"]:   # forward: x and the gates in, y out; backward: these and g in, gradients out
        return {"bytes": 11 * e * n, "flops": 110 * n}
    return {"bytes": 4 * e * n, "flops": 30 * n}


# ---------------------------------------------------------------- from the definitions, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    d = {k: (v.detach().double() if torch.is_tensor(v) and v.is_floating_point() else v)
         for k, v in s.items()}
    if case["op"] in ("addnorm", "norm8") and s["res"] is not None:
        # the stream holds its sum in its own type: that rounding is part of the definition
        d["res"] = (s["branch"].detach() + s["res"].detach()).to(s["res"].dtype).double()
    with torch.no_grad():
        return {"addnorm": _addnorm_exact, "norm8": _norm8_exact, "gated": _gated_exact,
                "token": _token_exact, "q4": _q4_exact}[case["op"]](d)


def _addnorm_exact(d):
    keep, w = d["res"], d["w"]
    n = keep.shape[1]
    norm = (torch.einsum("rd,rd->r", keep, keep) / n + d["eps"]).sqrt()[:, None]
    out = {"y": keep / norm * w, "s": keep}
    if d["grad"]:
        along = torch.einsum("rd,rd,d->r", d["gy"], keep, w)[:, None] / n
        ds = d["gs"] + d["gy"] * w / norm - keep * along / norm ** 3
        out.update(dx=ds, dres=ds, dw=torch.einsum("rd,rd->d", d["gy"], keep / norm))
    return out


def _norm8_exact(d):
    v = d["branch"] if d["res"] is None else d["res"]
    y = v / (torch.einsum("rd,rd->r", v, v) / v.shape[1] + d["eps"]).sqrt()[:, None] * d["w"]
    width = d["group"] or v.shape[1]
    scale = torch.stack([p.abs().max(1).values for p in y.split(width, dim=1)], 1) / 448
    out = {"q": y / scale.repeat_interleave(width, dim=1), "scale": scale}
    if d["res"] is not None:
        out["s"] = d["res"]
    return out


def _log_a(d):
    return -8.0 * torch.nn.functional.softplus(d["decay"], threshold=40) * torch.sigmoid(d["rg"])


def _gated_exact(d):
    x, g = d["x"], d["g"]
    B, L, D = x.shape
    r, i, l = torch.sigmoid(d["rg"]), torch.sigmoid(d["ig"]), _log_a(d)
    a = l.exp()
    m = (-torch.expm1(2 * l)).sqrt()
    n = d["lengths"].tolist() if d["lengths"] is not None else [L] * B
    h = d["state"].clone() if d["state"] is not None else x.new_zeros(B, D)
    live = torch.tensor([[t < k for t in range(L)] for k in n], device=x.device)[..., None]
    a, b = torch.where(live, a, 1.0), torch.where(live, m * i * x, 0.0)
    kept = torch.empty(L + 1, B, D, dtype=torch.float64, device=x.device)
    kept[0] = h
    for t in range(L):
        torch.addcmul(b[:, t], a[:, t], kept[t], out=kept[t + 1])
    y = kept[1:].transpose(0, 1) * live
    if g is None:
        return {"y": y, "state": kept[L].clone()}
    q = torch.empty_like(kept)
    q[L] = 0
    g = g * live
    for t in range(L - 1, -1, -1):
        after = a[:, t + 1] if t + 1 < L else torch.zeros_like(h)
        torch.addcmul(g[:, t], after, q[t + 1], out=q[t])
    q = q[:L].transpose(0, 1) * live
    da = q * kept[:L].transpose(0, 1)            # through the state
    dm = q * i * x                               # through the input's factor
    dl = da * a - dm * a * a / m
    out = {"y": y, "dx": q * m * i, "dig": q * m * x * i * (1 - i), "drg": dl * l * (1 - r)}
    sp = torch.nn.functional.softplus(d["decay"], threshold=40)
    out["ddecay"] = torch.einsum("bld,bld->d", dl, l) / sp * torch.sigmoid(d["decay"])
    return out


def _token_exact(d):
    l = _log_a(d)
    h = l.exp() * d["h"] + (-torch.expm1(2 * l)).sqrt() * torch.sigmoid(d["ig"]) * d["x"]
    return {"y": h, "h": h}


def _q4_exact(d):
    x, p, K = d["x"], d["packed"].long(), d["K"]
    if d["norm_w"] is not None:
        x = x / (torch.einsum("rk,rk->r", x, x) / K + d["eps"]).sqrt()[:, None] * d["norm_w"]
    y = torch.zeros(x.shape[0], d["N"], dtype=torch.float64, device=x.device)
    for j in range(d["scale"].shape[1]):         # a group of columns at a time
        lo, hi = j * d["group"], min(K, (j + 1) * d["group"])
        b = p[:, lo // 2:(hi + 1) // 2]
        codes = torch.empty(b.shape[0], 2 * b.shape[1], dtype=torch.float64, device=x.device)
        codes[:, 0::2], codes[:, 1::2] = b % 16, b // 16
        y += torch.einsum("rk,nk->rn", x[:, lo:hi], codes[:, :hi - lo] - 8) * d["scale"][:, j]
        if d["mid"] is not None:
            y += x[:, lo:hi].sum(1)[:, None] * d["mid"][:, j]
    y += d["bias"]
    if not d["split"]:
        return {"y": y}
    u = y[:, :d["cut"]]
    return {"u": u / (1 + (-u).exp()), "z": y[:, d["cut"]:]}
