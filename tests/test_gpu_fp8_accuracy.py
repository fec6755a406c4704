"""Dense products in 8 bits: how far results are off in all, beside what a single one may be at worst."""
from __future__ import annotations

import pytest
import torch

import fp8_exact as X
from test_gpu_fp8 import BF16_HALF, check, give, weight

pytestmark = pytest.mark.gpu

# The norm of a rounding to BF16 is 1.66e-3 of that of normal numbers (2^-7 / sqrt(28) of numbers evenly spread between powers of two, 2^-8 / sqrt(3) just above one),
# for 2048 and more of them within 3 % of it.  Scales that lost bits, 2^-9 each, would make 2.3e-3 of it.
BF16_NORM = 1.85e-3
# The instruction on the codes is 1.5e-5 of the norm off on normal operands, 1.2e-5 on the mean: 1.2e-5 over the distance between BF16 numbers of the results are
# carried to the next one, 1.5e-3 of those above the norm, twice as many of each power of two below until all of them are, in all 1.4 %.  Twice that loss
# doubles it.
NOT_NEAREST = 0.03


def normal(R, K, T, seed):
    """Codes as a normal matrix has them, and rows of normal activations."""
    g = torch.Generator().manual_seed(seed)
    codes = (torch.randn((R, K), generator=g) * 112).clamp_(-448, 448).to(X.E4M3)
    scales = (0.5 + torch.rand((-(-R // 128), -(-K // 128)), generator=g)) * 2e-4
    return codes, scales, torch.randn((T, K), generator=g)


@pytest.mark.parametrize("R,K,T", [(2048, 2048, 300), (520, 1040, 300), (1453, 2576, 140), (9000, 640, 3), (2000, 512, 2048)])
def test_many_columns(ops, R, K, T):
    c, s, x = normal(R, K, T, R)
    x, q, xs = give(x, "rows")
    y = X.product(q, xs, c, s)[0]
    w = weight(ops, c, s)
    got = ops.fp8_linear(x, w).cpu()
    assert ops.last_kernel().startswith("k_fp8_many") and (got.double() - y).norm() <= BF16_NORM * y.norm()
    assert (got != y.to(torch.bfloat16)).double().mean() <= NOT_NEAREST
    # FP32: a step for each block's sum, four for its products and scales
    got = ops.fp8_linear(x, w, out_dtype=torch.float32).cpu()
    assert (got.double() - y).norm() <= (-(-K // 128) + 4) * 2.0 ** -24 * y.norm()
    gate = ops.fp8_linear_glu2(x, w, w).cpu()
    want = y * torch.sigmoid(y) * y
    assert (gate.double() - want).norm() <= (2.0 ** -8 / 3 ** 0.5 + 4 * 1.5e-5) * want.norm()  # (its numbers are no normal ones; silu(y) y changes as y^2 does)


@pytest.mark.parametrize("R,K,T", [(512, 2048, 1), (512, 2048, 17), (300, 9104, 7), (400, 8192, 31), (1408, 2048, 64), (520, 1040, 100), (1453, 2576, 40), (4096, 512, 16)])
@pytest.mark.parametrize("kind", ["bf16", "f32", "rows"])
def test_few_columns_are_summed_exactly_whatever_the_result(ops, R, K, T, kind):
    """Operands of every size: FP32's bound and the result's rounding, nothing for what the instruction on the codes drops."""
    c, s = X.matrix(R, K, R + T)
    x, q, xs = give(X.rows(T, K, T), kind)
    y, dy = X.product(q, xs, c, s)
    got = ops.fp8_linear(x, weight(ops, c, s))
    assert ops.last_kernel().startswith("k_fp8_few")
    check(got, y, dy)
    g, dg = X.gated(y, dy, y, dy)
    got = ops.fp8_linear_glu2(x, weight(ops, c, s), weight(ops, c, s)).cpu().double()
    assert ((got - g).abs() <= dg + (g.abs() + dg) * BF16_HALF).all()
