"""Drawing tokens (a search's moves) from logits on the sm_100a kernels.

``m3_sample`` draws one token per row with temperature, top-k, top-p and min-p
from given uniform numbers: no random state of its own, so a rollout is a
function of its inputs.  There is no CPU path: it raises on CPU tensors.
"""

import torch

from . import _lib
from . import _launch as H
from ._lib import SampleDesc

MAX_VOCAB = 262144


def _setting(name, v, lead, dtype, lo, hi):
    """(array or None, scalar) of a setting given as one number or one per row; a
    number on the GPU stays there, as one per row, and is not waited for."""
    whole = torch.is_tensor(v) and not (v.dtype.is_floating_point or v.dtype is torch.bool)
    if torch.is_tensor(v) and (v.dim() or (v.is_cuda and (whole or dtype is not torch.int32))):
        if v.dim() == 0:
            v = v.expand(lead)
        if v.shape != lead:
            raise ValueError(f"m3_sample: {name} is a number or one per row")
        if dtype is torch.int32 and v.dtype is not dtype:
            if not whole:
                raise ValueError(f"m3_sample: {name} per row is a tensor of integers")
            v = v.to(torch.int64).clamp(0, 2 ** 31 - 1)
        return (v if v.dtype is dtype else v.detach().to(dtype)).contiguous(), 0
    v = float(v)
    if not lo <= v <= hi or (dtype is torch.int32 and v != int(v)):
        raise ValueError(f"m3_sample: {name} must lie in [{lo}, {hi}]"
                         + (" and be whole" if dtype is torch.int32 else ""))
    return None, v


def m3_sample(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Tokens (int64) drawn from ``logits`` (V,) or (rows, V), float32 or bfloat16.

    With w = exp((logit - max) / temperature) over the candidates -- logits of
    -infinity (moves that are not allowed) and NaN are none -- ordered by logit,
    equal ones by index: ``top_k`` keeps the first k (0: all); ``top_p``, of
    those, the shortest prefix with at least that share of their weight, one
    token at least (1: all); ``min_p``, of those, the tokens with w >= min_p.
    The token is the smallest index whose cumulative weight over the kept tokens,
    in index order, exceeds ``uniform`` (one number in [0, 1) per row, float32)
    times their total.  Temperature 0 takes the largest logit, the lowest index
    among equals.  A row without candidates gives -1.

    Each setting is a number (rounded to float32), or a tensor of one per row or,
    0-dim, of one for all (float32; integers for top_k).  Values in tensors on the
    GPU are not checked: a temperature that is negative or NaN counts as 0, top_k
    below 0 as 0, top_p that is NaN or below 0 as 0, min_p above 1 or NaN as 1.
    V <= 262144."""
    if logits.dim() not in (1, 2) or logits.shape[-1] < 1:
        raise ValueError("m3_sample: logits are (V,) or (rows, V)")
    V, lead = logits.shape[-1], logits.shape[:-1]
    if V > MAX_VOCAB:
        raise ValueError(f"m3_sample: at most {MAX_VOCAB} logits per row")
    if lead:
        H.check_sizes("m3_sample", lead[0])
    if uniform.shape != lead or uniform.dtype != torch.float32:
        raise ValueError("m3_sample: uniform is float32, one number per row")
    code = H.code(logits.dtype)
    t, t0 = _setting("temperature", temperature, lead, torch.float32, 0.0, float("inf"))
    k, k0 = _setting("top_k", top_k, lead, torch.int32, 0, 2 ** 31 - 1)
    p, p0 = _setting("top_p", top_p, lead, torch.float32, 0.0, 1.0)
    m, m0 = _setting("min_p", min_p, lead, torch.float32, 0.0, 1.0)
    dev = H.device_index(logits, uniform, t, k, p, m)
    rows = lead[0] if lead else 1
    out = torch.empty(lead, device=logits.device, dtype=torch.int64)
    if rows == 0:
        return out
    x, ld = H.rows(logits if lead else logits.unsqueeze(0))
    u = uniform.contiguous()
    H.launch(dev, _lib.load().m3_sample, SampleDesc(rows, V, code, t0, int(k0), p0, m0),
             x.data_ptr(), ld, u.data_ptr(), H.ptr(t), H.ptr(k), H.ptr(p), H.ptr(m),
             out.data_ptr())
    return out
