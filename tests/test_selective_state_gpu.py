"""The states of the convolution and the scan between training and tokens."""

import pytest
import torch

from redpanda_b200 import selective as S

pytestmark = pytest.mark.gpu


def _inputs():
    g = torch.Generator().manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    return r(2, 9, 24), r(24, 4), r(2, 9, 24), -r(24, 8).abs(), r(2, 9, 8), r(2, 9, 8)


def test_a_step_between_forward_and_backward_is_noticed():
    """A step writes its state in place; a backward pass that has saved the same
    state raises, as after any in-place operation, instead of using the new one."""
    x, w, dt, A, b, c = _inputs()
    w.requires_grad_(True)
    state = torch.zeros(2, 3, 24, device="cuda")
    y = S.m3_causal_conv(x, w, state=state)
    ref = torch.autograd.grad(y.sum(), w, retain_graph=True)[0]
    with torch.no_grad():
        S.m3_causal_conv_step_(state.clone(), x[:, 0], w)        # another tensor: no harm
    assert torch.equal(torch.autograd.grad(y.sum(), w, retain_graph=True)[0], ref)
    with torch.no_grad():
        S.m3_causal_conv_step_(state, x[:, 0], w)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y.sum(), w)

    A.requires_grad_(True)
    h = torch.zeros(2, 24, 8, device="cuda")
    y = S.m3_selective_scan(x, dt, A, b, c, state=h)
    with torch.no_grad():
        S.m3_selective_step_(h, x[:, 0], dt[:, 0], A, b[:, 0], c[:, 0])
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y.sum(), A)


def test_steps_work_under_inference_mode():
    x, w, dt, A, b, c = _inputs()
    s0, h0 = torch.zeros(2, 3, 24, device="cuda"), torch.zeros(2, 24, 8, device="cuda")
    ref = (S.m3_causal_conv_step_(s0, x[:, 0], w),
           S.m3_selective_step_(h0, x[:, 0], dt[:, 0], A, b[:, 0], c[:, 0]))
    with torch.inference_mode():
        s1, h1 = torch.zeros(2, 3, 24, device="cuda"), torch.zeros(2, 24, 8, device="cuda")
        got = (S.m3_causal_conv_step_(s1, x[:, 0], w),
               S.m3_selective_step_(h1, x[:, 0], dt[:, 0], A, b[:, 0], c[:, 0]))
    for p, q in zip((*ref, s0, h0), (*got, s1, h1)):
        assert torch.equal(p, q)
