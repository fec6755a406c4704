"""The low bits of FP32 activations and of the zero points' product: inputs for which only the third of the three BF16 parts is left, or
whose results are bounded by a few FP32 steps of themselves.

Bounds.  A product of a code (4 bits) or of a part (8 bits) with a part is exact in FP32.
  cancel   v and -(v without its third part l), equal codes u, one group: the first and second parts' sums are exactly zero whatever the
           order, the third's is u l, the activations' sum l; fma(-z, l, u l) is exact ((u - z) l has at most 16 bits) and the scaled one is
           rounded once: half a step, 2^-24 |y|.
  single   one activation v that is not zero: two additions of the parts' sums, relative to u |v|, and two fused ones, relative to
           |u - z| |v|: half a step, 2^-24, each.
  zeros    many columns, all codes zero, one group of a token not zero: y = -s z X with X exact (24 bits by construction).  Eight exact
           products and eight additions of the matrix cores, a whole step, 2^-23, each, of partial sums that are no more than 1 + 2^-6 times
           |s z X|; X3 Z3 left out, 2^-28.  What is added behind that is zero."""
from __future__ import annotations

import pytest
import torch

import int4_exact as X

pytestmark = pytest.mark.gpu


def matrix(ops, rows, K, group, seed, zeros, f16=False):
    m = X.make(rows, K, group, seed, zeros, f16)
    return m, lambda codes: ops.Int4Weight(codes.cuda(), m[1].cuda(), None if m[2] is None else m[2].cuda(), group)


def packed(u):
    u = u.to(torch.uint8)
    return u[:, 0::2] | (u[:, 1::2] << 4)


# 24 bits with ones in the last eight, signs and exponents apart
VALUES = [1.0 + 2.0 ** -4 + 2.0 ** -11 + 171 * 2.0 ** -23, -(1.5 + 2.0 ** -9 + 255 * 2.0 ** -23) * 2.0 ** 20, (1.25 + 2.0 ** -10 + 129 * 2.0 ** -23) * 2.0 ** -30]


@pytest.mark.parametrize("rows,K", [(48, 352), (9000, 352), (40, 2048), (9000, 96)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [True, False])
def test_third_part_of_an_activation(ops, rows, K, group, zeros):
    m, of = matrix(ops, rows, K, group, rows + K + group, zeros)
    u, s, z = X.parts(*m, group)
    for a, b in ((0, 1), (5, 17), (K - 32, K - 1), (33, 64 - 1)):
        x = torch.zeros((len(VALUES), K))
        x[:, a] = torch.tensor(VALUES)
        assert torch.equal(x[:, a].double(), torch.tensor(VALUES, dtype=torch.float64))
        high = x[:, a].view(torch.int32).bitwise_and(~0xFF).view(torch.float32)  # (sixteen leading bits: two parts)
        third = (x[:, a] - high).double()
        assert bool((third != 0).all())
        got = ops.int4_mmv(x.cuda(), of(m[0]))
        y = x[:, a].double()[:, None] * (s * (u - z))[:, a]
        bound = x[:, a].double().abs()[:, None] * (s.abs() * (u + (u - z).abs()))[:, a] * 2.0 ** -23
        X.check(got, y, bound * 1.001 + 1e-37, ("single", a))
        x[:, b] = -high
        ub = u.clone()
        ub[:, b] = ub[:, a]
        got = ops.int4_mmv(x.cuda(), of(packed(ub)))
        y = third[:, None] * (s * (u - z))[:, a]
        X.check(got, y, 2.0 ** -24 * y.abs() * 1.001 + 1e-37, ("cancel", a, b))


@pytest.mark.parametrize("rows,K,T,group", [(8300, 416, 70, 32), (8300, 544, 70, 32), (8300, 832, 70, 64), (8300, 1056, 70, 128)])
@pytest.mark.parametrize("f16", [False, True])
def test_parts_of_the_zero_points_product(ops, rows, K, T, group, f16):
    m, of = matrix(ops, rows, K, group, K, True, f16)
    g = torch.Generator().manual_seed(T)
    n = -(-K // group)
    x = torch.zeros((T, K))
    for t in range(T):
        first = t % n * group  # (the last group may be cut short)
        at = first + torch.randperm(min(group, K - first), generator=g)[:3]
        one, two, three = (int(v) for v in torch.randint(128, 256, (3,), generator=g))
        x[t, at] = torch.tensor([one * 2.0 ** -7, (two | 1) * 2.0 ** -15, (three | 1) * 2.0 ** -23]) * (-1.0) ** t
    xb = x.to(torch.bfloat16)
    assert torch.equal(xb.float(), x)
    total = torch.stack([p.double().sum(1) for p in x.split(group, 1)], 1)
    assert torch.equal(total.float().double(), total)
    got = ops.int4_mmv(xb.cuda(), of(torch.zeros_like(m[0])))
    y = -(total @ (m[1].double() * m[2].double()).t())
    X.check(got, y, y.abs() * (8 * 1.016 * 2.0 ** -23 + 2.0 ** -28))
