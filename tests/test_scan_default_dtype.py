"""Buffers of the trapezoidal scan under another default element type of torch's:
the kernels read and write float32 in them."""

import contextlib

import pytest
import torch

from redpanda_b200 import scan as S
from redpanda_b200.mamba import Mamba3Block, MambaConfig
from test_default_dtype import _default


class _Library:
    """Stands for the library on the host: sizes, and entries that return 0."""
    def __getattr__(self, name):
        return lambda *a: 64 if name.endswith(("_floats", "_bytes")) else 0


def _on_the_host(monkeypatch):
    monkeypatch.setattr(S, "_require_cuda", lambda *ts: torch.device("cpu"))
    monkeypatch.setattr(S, "_stream", lambda dev: 0)
    monkeypatch.setattr(S._lib, "load", lambda: _Library())
    monkeypatch.setattr(S._lib, "check", lambda rc: None)
    monkeypatch.setattr(torch.cuda, "device", lambda dev: contextlib.nullcontext())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float64])
def test_fused_scan_checkpoints_are_float32(dtype, monkeypatch):
    _on_the_host(monkeypatch)
    bf = lambda *s: torch.ones(*s, dtype=torch.bfloat16)  # noqa: E731
    dt, x, u = bf(2, 20, 8), bf(2, 20, 20), bf(2, 20, 8).requires_grad_(True)
    A = torch.ones(8, 4, dtype=torch.float32)
    with _default(dtype):
        y = S.m3_fused_scan(dt, x, None, None, 1e-5, u, A, A, None, 4, 4, 2, 0, 8)
    ckpt = y.grad_fn.saved_tensors[6]
    assert ckpt.numel() == 64 and ckpt.dtype == torch.float32


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float64])
def test_padded_parameters_and_states_are_float32(dtype, monkeypatch):
    A = torch.ones(8, 4, dtype=torch.float32)
    with _default(dtype):
        for args in ((A, None, None), (None, None, A), (A, A, None)):
            assert {t.dtype for t in S.pad_params(*args, 4, 8, 8, "cpu")} == {torch.float32}
        block = Mamba3Block(MambaConfig(d_model=8, n_layer=1, d_state=8, n_track_state=0, mimo_p=1))
        monkeypatch.setattr(block, "step_", lambda x, state: state)
        assert {t.dtype for t in block.step(torch.zeros(3, 8))} == {torch.float32}
