"""Derivatives that the sequence-model operators do not have are refused, on the
host, before any launch."""

import pytest
import torch
from torch.autograd import forward_ad

from redpanda_b200 import norm as N
from redpanda_b200 import selective as S

z = torch.zeros

CALLS = {
    "m3_layer_norm": (N.m3_layer_norm, lambda: [z(2, 8), z(8), z(8)]),
    "m3_rms_norm": (N.m3_rms_norm, lambda: [z(2, 8), z(8)]),
    "m3_causal_conv": (S.m3_causal_conv, lambda: [z(1, 4, 8), z(8, 4), z(8)]),
    "m3_causal_conv_with_state": (S.m3_causal_conv_with_state, lambda: [z(1, 4, 8), z(8, 4)]),
    "m3_causal_conv_step_": (S.m3_causal_conv_step_, lambda: [z(1, 3, 8), z(1, 8), z(8, 4)]),
    "m3_selective_scan": (S.m3_selective_scan, lambda: [
        z(1, 4, 8), z(1, 4, 8), z(8, 2), z(1, 4, 2), z(1, 4, 2), z(8), z(1, 4, 8), z(8)]),
    "m3_selective_scan_with_state": (S.m3_selective_scan_with_state, lambda: [
        z(1, 4, 8), z(1, 4, 8), z(8, 2), z(1, 4, 2), z(1, 4, 2)]),
    "m3_selective_step_": (S.m3_selective_step_, lambda: [
        z(1, 8, 2), z(1, 8), z(1, 8), z(8, 2), z(1, 2), z(1, 2), z(8), z(1, 8), z(8)]),
}


@pytest.mark.parametrize("name", CALLS)
def test_forward_mode_tangents_are_refused(name):
    """A dual tensor in any place, with gradients on and off; none is dropped."""
    fn, make = CALLS[name]
    for i in range(len(make())):
        with forward_ad.dual_level():
            a = make()
            a[i] = forward_ad.make_dual(a[i], torch.ones_like(a[i]))
            with pytest.raises(ValueError, match="forward-mode"):
                fn(*a)
            with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
                fn(*a)
            # a level without a dual tensor changes nothing: CPU tensors are refused
            with pytest.raises(RuntimeError, match="CUDA"):
                fn(*make())
        with pytest.raises(RuntimeError, match="CUDA"):
            fn(*make())


def test_tangents_of_states_are_refused():
    with forward_ad.dual_level():
        st = forward_ad.make_dual(z(1, 3, 8), torch.ones(1, 3, 8))
        with pytest.raises(ValueError, match="forward-mode"):
            S.m3_causal_conv(z(1, 4, 8), z(8, 4), state=st)
        h = forward_ad.make_dual(z(1, 8, 2), torch.ones(1, 8, 2))
        with pytest.raises(ValueError, match="forward-mode"):
            S.m3_selective_scan(z(1, 4, 8), z(1, 4, 8), z(8, 2), z(1, 4, 2), z(1, 4, 2), state=h)
