"""The 4-bit weight's layout and rounding, on the CPU, and what it refuses."""

import pytest
import torch

from redpanda_b200 import quant as Q

z = torch.zeros


def made(n, k, group, center, seed=0):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (n, k), generator=g)
    ng = -(-k // group)
    scale = torch.rand(n, ng, generator=g).add_(0.1).bfloat16()
    mid = torch.randn(n, ng, generator=g).bfloat16() if center else None
    wide = scale.float().repeat_interleave(group, 1)[:, :k]
    w = (codes - 8).float() * wide
    if center:
        w = w + mid.float().repeat_interleave(group, 1)[:, :k]
    return codes, scale, mid, w


SHAPES = [(5, 33, 32), (40, 300, 64), (17, 129, 128), (1, 1, 32), (33, 64, 64), (16, 7, 128)]


@pytest.mark.parametrize("center", [False, True])
@pytest.mark.parametrize("n,k,group", SHAPES)
def test_layout_and_back(n, k, group, center):
    codes, scale, mid, w = made(n, k, group, center)
    q = Q.Q4Weight.from_codes(codes, scale, mid, group)
    # an fp32 product and sum of bf16 scale and center: the same operations, the same bits
    assert torch.equal(q.dequantize(), w)
    pad = torch.nn.functional.pad(codes, (0, k & 1)).to(torch.uint8)
    p = Q.Q4Weight.from_packed(pad[:, ::2] | pad[:, 1::2] << 4, scale, mid, k, group)
    assert torch.equal(p.codes, q.codes) and torch.equal(p.scales, q.scales)
    # the words as the header states them
    blocks = q.codes.shape[1]
    for o in range(n):
        for c in range(k):
            word = int(q.codes[o // 16, c // 64, (o % 8) * 4 + c % 32 // 8,
                               c % 64 // 32 * 2 + c % 8 // 4])
            at = 4 * (o % 16 // 8 + 2 * (c % 4 // 2) + 4 * (c % 2))
            assert (word >> at) & 15 == codes[o, c]
    assert blocks * 64 % max(group, 64) == 0


@pytest.mark.parametrize("center", [False, True])
@pytest.mark.parametrize("n,k,group", SHAPES)
def test_quantize_is_near(n, k, group, center):
    w = torch.randn(n, k, generator=torch.Generator().manual_seed(n + k))
    q = Q.Q4Weight.quantize(w, group, center)
    wide = torch.nn.functional.pad(w, (0, -k % group)).view(n, -1, group)
    real = torch.arange(wide.shape[1] * group).view(1, -1, group) < k
    lo = torch.where(real, wide, torch.inf).amin(2)
    hi = torch.where(real, wide, -torch.inf).amax(2)
    step = ((hi - lo) / 15 if center else torch.maximum(hi / 7, -lo / 8))
    # half a step; the bf16 scale is 2^-8 off over up to 15 steps (from the center 8), the
    # center by 2^-8 of itself, whose size is below |lo| + 8 steps
    size = torch.maximum(lo.abs(), hi.abs())
    tol = step * (0.5 + 15 * 2.0 ** -8) + (size + 8 * step) * 2.0 ** -8 + 1e-6
    far = (q.dequantize() - w).abs()
    assert (far <= tol.repeat_interleave(group, 1)[:, :k]).all()


def test_quantize_of_the_largest_weights():
    """A range that overflows as a difference."""
    w = torch.tensor([[-3e38, 3e38, 1e38, 0.0]])
    back = Q.Q4Weight.quantize(w, 32).dequantize()
    # a code's step is 4e37, its scale and center 2^-8 off
    assert torch.isfinite(back).all() and ((back - w).abs() <= 2e37 + 15 * 4e37 / 256 + 3e38 / 256).all()


def test_quantize_of_constant_groups():
    w = torch.full((3, 64), 0.75)
    w[1] = 0
    q = Q.Q4Weight.quantize(w)
    assert torch.equal(q.dequantize(), w)
    assert not Q.Q4Weight.quantize(z(2, 40), 32, center=False).dequantize().any()


@pytest.mark.parametrize("call", [
    lambda: Q.Q4Weight.quantize(z(4, 64), group=48),
    lambda: Q.Q4Weight.quantize(z(4)),
    lambda: Q.Q4Weight.quantize(z(0, 4)),
    lambda: Q.Q4Weight.quantize(z(1, 65537)),
    lambda: Q.Q4Weight.quantize(torch.tensor([[1.0, float("nan")]])),
    lambda: Q.Q4Weight.quantize(torch.tensor([[1.0, float("-inf")]])),
    lambda: Q.Q4Weight.from_codes(z(4, 64).int() + 16, z(4, 1)),
    lambda: Q.Q4Weight.from_codes(z(4, 64).int() - 1, z(4, 1)),
    lambda: Q.Q4Weight.from_codes(z(4, 64).int(), z(4, 2)),
    lambda: Q.Q4Weight.from_codes(z(4, 64).int(), z(4, 1).int()),
    lambda: Q.Q4Weight.from_codes(z(4, 64).int(), z(4, 1), z(1, 4)),
    lambda: Q.Q4Weight.from_packed(z(4, 32).byte(), z(4, 1), d_in=62),
    lambda: Q.Q4Weight.from_packed(z(4, 32).int(), z(4, 1)),
])
def test_weights_that_are_refused(call):
    with pytest.raises(ValueError):
        call()


def test_codes_of_another_type_are_refused():
    for t in (torch.float32, torch.bool):
        with pytest.raises(TypeError):
            Q.Q4Weight.from_codes(z(4, 64, dtype=t), z(4, 1))


W = Q.Q4Weight.quantize(torch.ones(6, 40), 32)


@pytest.mark.parametrize("call", [
    lambda: Q.m3_rows_linear_q4(z(9, 40), W),
    lambda: Q.m3_rows_linear_q4(z(2, 41), W),
    lambda: Q.m3_rows_linear_q4(z(40), W),
    lambda: Q.m3_rows_linear_q4(z(2, 40), W, z(7)),
    lambda: Q.m3_rows_linear_q4(z(2, 40), W, norm_weight=z(6)),
    lambda: Q.m3_rows_linear_q4(z(2, 40), W, eps=-1.0),
    lambda: Q.m3_rows_linear_q4(z(2, 40), W, split=7),
    lambda: Q.m3_rows_linear_q4(z(2, 40), W, bias=z(6).requires_grad_(True)),
])
def test_products_that_are_refused(call):
    with pytest.raises(ValueError):
        call()


def test_no_cpu_product_and_no_other_types():
    with pytest.raises(RuntimeError, match="CUDA"):
        Q.m3_rows_linear_q4(z(2, 40), W)
    with pytest.raises(TypeError):
        Q.m3_rows_linear_q4(z(2, 40).half(), W)
    with pytest.raises(TypeError):
        Q.m3_rows_linear_q4(z(2, 40), z(6, 40))
