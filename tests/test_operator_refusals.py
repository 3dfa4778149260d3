"""What the sequence-model operators refuse, on the host, before any launch."""

import ctypes

import pytest
import torch

from redpanda_b200 import _lib
from redpanda_b200 import norm as N
from redpanda_b200 import selective as S
from redpanda_b200.sampling import m3_sample

z = torch.zeros


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CUDA"):
        N.m3_layer_norm(z(2, 8), z(8))
    with pytest.raises(RuntimeError, match="CUDA"):
        S.m3_causal_conv(z(1, 4, 8), z(8, 4))
    with pytest.raises(RuntimeError, match="CUDA"):
        S.m3_causal_conv_step_(z(1, 3, 8), z(1, 8), z(8, 4))
    with pytest.raises(RuntimeError, match="CUDA"):
        S.m3_selective_scan(z(1, 4, 8), z(1, 4, 8), z(8, 2), z(1, 4, 2), z(1, 4, 2))
    with pytest.raises(RuntimeError, match="CUDA"):
        S.m3_selective_step_(z(1, 8, 2), z(1, 8), z(1, 8), z(8, 2), z(1, 2), z(1, 2))
    with pytest.raises(RuntimeError, match="CUDA"):
        m3_sample(z(2, 8), z(2))


@pytest.mark.parametrize("call", [
    lambda: N.m3_layer_norm(z(2, 8), z(7)),
    lambda: N.m3_layer_norm(z(2, 8), z(8), z(9)),
    lambda: N.m3_layer_norm(z(2, 0), z(0)),
    lambda: N.m3_rms_norm(z(2, 8), z(8), eps=-1.0),
    lambda: N.m3_rms_norm(z(2, 8), z(8), eps=float("nan")),
    lambda: N.m3_rms_norm(z(1, 40000), z(40000)),
    lambda: S.m3_causal_conv(z(4, 8), z(8, 4)),
    lambda: S.m3_causal_conv(z(1, 4, 8), z(8, 9)),
    lambda: S.m3_causal_conv(z(1, 4, 8), z(7, 4)),
    lambda: S.m3_causal_conv(z(1, 4, 8), z(8, 4), z(4)),
    lambda: S.m3_causal_conv(z(1, 4, 8), z(8, 4), state=z(1, 4, 8)),
    lambda: S.m3_causal_conv(z(1, 4, 8), z(8, 4), state=z(1, 3, 8).bfloat16()),
    lambda: S.m3_causal_conv(z(2, 4, 8), z(8, 4), lengths=z(1, dtype=torch.int32)),
    lambda: S.m3_causal_conv(z(2, 4, 8), z(8, 4), lengths=z(2)),
    lambda: S.m3_causal_conv_step_(z(1, 2, 8), z(1, 8), z(8, 4)),
    lambda: S.m3_selective_scan(z(1, 4, 8), z(1, 4, 7), z(8, 2), z(1, 4, 2), z(1, 4, 2)),
    lambda: S.m3_selective_scan(z(1, 4, 8), z(1, 4, 8), z(8, 2), z(1, 4, 3), z(1, 4, 2)),
    lambda: S.m3_selective_scan(z(1, 4, 8), z(1, 4, 8), z(8, 129), z(1, 4, 129), z(1, 4, 129)),
    lambda: S.m3_selective_scan(z(1, 4, 8), z(1, 4, 8), z(8, 2), z(1, 4, 2), z(1, 4, 2), D=z(7)),
    lambda: S.m3_selective_scan(z(1, 4, 8), z(1, 4, 8), z(8, 2), z(1, 4, 2), z(1, 4, 2),
                                z=z(1, 3, 8)),
    lambda: S.m3_selective_scan(z(1, 4, 8), z(1, 4, 8), z(8, 2), z(1, 4, 2), z(1, 4, 2),
                                state=z(1, 8, 3)),
    lambda: S.m3_selective_step_(z(1, 8, 3), z(1, 8), z(1, 8), z(8, 2), z(1, 2), z(1, 2)),
    lambda: S.m3_selective_step_(z(1, 8, 2).double(), z(1, 8), z(1, 8), z(8, 2), z(1, 2), z(1, 2)),
    lambda: m3_sample(z(2, 3, 4), z(2)),
    lambda: m3_sample(z(2, 8), z(3)),
    lambda: m3_sample(z(2, 8), z(2).double()),
    lambda: m3_sample(z(2, 8), z(2), temperature=-0.5),
    lambda: m3_sample(z(2, 8), z(2), temperature=float("nan")),
    lambda: m3_sample(z(2, 8), z(2), top_p=1.5),
    lambda: m3_sample(z(2, 8), z(2), min_p=-0.1),
    lambda: m3_sample(z(2, 8), z(2), top_k=-1),
    lambda: m3_sample(z(2, 8), z(2), top_k=2.5),
    lambda: m3_sample(z(2, 8), z(2), top_k=z(3, dtype=torch.int32)),
    lambda: m3_sample(z(2, 8), z(2), top_k=z(2)),
    # sizes that 32 bits would cut short
    lambda: m3_sample(z(1, 1).expand(2 ** 32 + 1, 1), z(1).expand(2 ** 32 + 1)),
    lambda: S.m3_causal_conv(z(1, 1, 1).expand(1, 2 ** 32 + 5, 1), z(1, 1)),
    lambda: S.m3_causal_conv_step_(z(1, 0, 1).expand(2 ** 31, 0, 1),
                                   z(1, 1).expand(2 ** 31, 1), z(1, 1)),
    lambda: S.m3_selective_scan(*2 * [z(1, 1, 1).expand(1, 2 ** 32 + 5, 1)], z(1, 1),
                                *2 * [z(1, 1, 1).expand(1, 2 ** 32 + 5, 1)]),
    lambda: S.m3_selective_step_(z(1, 1, 1).expand(2 ** 31, 1, 1), *2 * [z(1, 1).expand(2 ** 31, 1)],
                                 z(1, 1), *2 * [z(1, 1).expand(2 ** 31, 1)]),
    lambda: m3_sample(z(1, 262145), z(1)),
])
def test_bad_arguments_raise_value_errors(call):
    with pytest.raises(ValueError):
        call()


@pytest.mark.parametrize("call", [
    lambda: N.m3_layer_norm(z(2, 8).half(), z(8)),
    lambda: N.m3_layer_norm(z(2, 8), z(8), out_dtype=torch.float64),
    lambda: S.m3_causal_conv(z(1, 4, 8).double(), z(8, 4)),
    lambda: S.m3_selective_scan(z(1, 4, 8).half(), z(1, 4, 8), z(8, 2), z(1, 4, 2), z(1, 4, 2)),
    lambda: m3_sample(z(2, 8).half(), z(2)),
])
def test_other_element_types_are_refused(call):
    with pytest.raises(TypeError):
        call()


def test_states_are_not_differentiable():
    with pytest.raises(ValueError, match="differentiable"):
        S.m3_causal_conv(z(1, 4, 8), z(8, 4), state=z(1, 3, 8, requires_grad=True))
    with pytest.raises(ValueError, match="no_grad"):
        S.m3_causal_conv_step_(z(1, 3, 8), z(1, 8, requires_grad=True), z(8, 4))


def test_c_entries_validate_before_device_work():
    """Status codes of bad descriptors and pointers (no device is touched)."""
    lib = _lib.load()
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) // 256 * 256     # host memory: never dereferenced
    n = None

    def norm(rows=2, d=8, tx=0, ty=0, rms=0, eps=1e-5, x=p, ld=8, w=p, y=p):
        return lib.m3_norm_fwd(_lib.NormDesc(rows, d, tx, ty, rms, eps), x, ld, w, n, y, n, n, n)
    assert lib.m3_norm_fwd(n, p, 8, p, n, p, n, n, n) == 1
    assert [norm(x=n), norm(w=n), norm(y=n)] == [1, 1, 1]
    assert [norm(rows=0), norm(d=0), norm(eps=-1.0), norm(ld=7)] == [2, 2, 2, 2]
    assert [norm(tx=5), norm(ty=-1), norm(d=40000, ld=40000), norm(x=p + 2)] == [3, 3, 4, 5]
    d = _lib.NormDesc(2, 8, 0, 0, 0, 1e-5)
    assert lib.m3_norm_bwd(d, p, 8, p, n, p, p, p, p, n, p, 4096, n) == 1     # no means

    def conv(B=1, L=4, D=8, K=4, ty=0, x=p, ld=8, st=n, y=p + 512, so=n):
        return lib.m3_causal_conv_fwd(_lib.ConvDesc(B, L, D, K, ty, 1), x, ld, p, n, st, n, y, so, n)
    assert [conv(B=0), conv(L=0), conv(D=0), conv(K=0), conv(ld=7)] == [2] * 5
    big = (1 << 30) + 1
    assert [conv(B=big), conv(L=big), conv(D=big, ld=big)] == [2] * 3
    assert [conv(K=9), conv(ty=2), conv(x=n), conv(x=p + 1)] == [4, 3, 1, 5]
    assert [conv(y=p), conv(st=p + 1024, so=p + 1024)] == [11, 11]
    c = _lib.ConvDesc(1, 4, 8, 4, 0, 1)
    assert lib.m3_causal_conv_step(c, p, p + 512, 8, p, n, p + 1024, n) == 2   # seqlen is 1
    c = _lib.ConvDesc(1, 1, 8, 4, 0, 1)
    assert lib.m3_causal_conv_step(c, n, p, 8, p, n, p + 512, n) == 1
    assert lib.m3_causal_conv_step(c, p, p, 8, p, n, p + 512, n) == 11

    def args(**kw):
        a = dict(u=p, u_ld=8, dt=p, dt_ld=8, z=n, z_ld=0, B=p, B_ld=2, C=p, C_ld=2, A=p)
        return _lib.SelArgs(**{**a, **kw})

    def sel(B=1, L=4, D=8, Ns=2, ty=0, a=None, y=p, h=n, ws=n, nws=0):
        return lib.m3_selective_fwd(_lib.SelDesc(B, L, D, Ns, ty, 1), a or args(), y, h, n, ws, nws, n)
    assert [sel(B=0), sel(L=0), sel(D=0), sel(Ns=0)] == [2] * 4
    assert [sel(L=big), sel(L=2 ** 31 - 1), sel(B=big),
            sel(D=2 ** 31 - 1, a=args(u_ld=2 ** 31, dt_ld=2 ** 31))] == [2] * 4
    assert [sel(ty=3), sel(Ns=129, a=args(B_ld=129, C_ld=129)), sel(y=n)] == [3, 4, 1]
    assert [sel(a=args(u=n)), sel(a=args(A=n)), sel(a=args(u_ld=7)), sel(a=args(B_ld=1)),
            sel(a=args(u=p + 2)), sel(a=args(z=p, z_ld=4))] == [1, 1, 2, 2, 5, 2]
    assert sel(a=args(state=p), h=p) == 11
    d1 = _lib.SelDesc(1, 1, 8, 2, 0, 1)
    assert lib.m3_selective_step(d1, args(state=p), p, p, n) == 4
    assert lib.m3_selective_step(d1, args(), n, p, n) == 1
    assert lib.m3_selective_step(_lib.SelDesc(1, 2, 8, 2, 0, 1), args(), p, p, n) == 2

    def sample(rows=1, V=8, ty=0, x=p, ld=8, u=p, out=p):
        return lib.m3_sample(_lib.SampleDesc(rows, V, ty, 1.0, 0, 1.0, 0.0), x, ld, u, n, n, n, n,
                             out, n)
    assert [sample(rows=0), sample(V=0), sample(ld=7), sample(ty=9)] == [2, 2, 2, 3]
    assert [sample(x=n), sample(u=n), sample(out=n), sample(out=p + 4)] == [1, 1, 1, 5]
    assert sample(V=1 << 19, ld=1 << 19) == 4


def test_checkpoint_sizes():
    lib = _lib.load()
    f = lambda **k: lib.m3_selective_ckpt_floats(  # noqa: E731
        _lib.SelDesc(*{**dict(B=2, L=16, D=8, N=16, ty=0, sp=1), **k}.values()))
    assert f() == 0 and f(L=17) == 2 * 8 * 16 and f(L=64, N=20) == 2 * 3 * 8 * 32
