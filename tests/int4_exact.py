"""4-bit weights with group scales in 64 bits, from the definition, with bounds of what the kernels' arithmetic may be off by.

A product of an exact code and a BF16 activation (or one of the three BF16 parts of an FP32 one) is exact in FP32; the
additions are not.  A term passes at most 128 of them within its 128 columns (the matrix cores may round an addition down
rather than to nearest: a whole step, 2^-23, each), two roundings per group and one per 128 columns further on, eight parts
of K, three parts of an FP32 activation; all relative to the sum of s * (u + z) * |x|, which bounds every partial sum."""
from __future__ import annotations

import torch

STEP32 = 2.0 ** -23
HALF_BF16 = torch.finfo(torch.bfloat16).eps / 2


def make(rows, K, group, seed, zeros=True, f16=False, device="cpu"):
    """(codes, scales, zeros or None) with codes over their whole range"""
    g = torch.Generator().manual_seed(seed)
    n = -(-K // group)
    codes = torch.randint(0, 256, (rows, K // 2), generator=g, dtype=torch.uint8)
    scales = ((0.5 + torch.rand((rows, n), generator=g)) * 0.01 * (torch.randint(0, 2, (rows, n), generator=g) * 2 - 1))
    z = torch.randint(0, 16, (rows, n), generator=g, dtype=torch.uint8) if zeros else None
    return codes.to(device), scales.to(torch.float16 if f16 else torch.bfloat16).to(device), None if z is None else z.to(device)


def parts(codes, scales, zeros, group):
    """(code, scale, zero) of every weight in 64 bits, on the CPU"""
    codes, scales = codes.cpu(), scales.cpu()
    u = torch.stack((codes & 15, codes >> 4), 2).flatten(1).double()
    of = torch.arange(u.shape[1]) // group
    z = torch.full_like(u, 8.0) if zeros is None else zeros.cpu().double()[:, of]
    return u, scales.double()[:, of], z


def product(x, w):
    """(y, bound) [tokens, rows] of x [tokens, K] and w = (codes, scales, zeros, group); bound without the rounding of the result"""
    u, s, z = parts(*w)
    x = x.cpu().double()
    y = x @ (s * (u - z)).t()
    K, group = u.shape[1], min(w[3], 128)
    depth = 128 + 3 * -(-K // group) + -(-K // 128) + 8 + 3
    return y, depth * STEP32 * (x.abs() @ (s.abs() * (u + z)).t()) + 1e-37


def gated(g, bg, u, bu):
    """(silu(g) * u, bound): |silu'| < 1.1; the exponential is off by (|g| + 8) steps of FP32, relative"""
    silu = g * torch.sigmoid(g)
    b = 1.1 * bg * (u.abs() + bu) + silu.abs() * bu + (silu * u).abs() * ((g.abs() + 8) * STEP32)
    return silu * u, b + 1e-37


def rounded(y, bound, dtype):
    return bound if dtype is torch.float32 else bound + HALF_BF16 * (y.abs() + bound)


def check(got, y, bound, what=""):
    err = (got.cpu().double() - y).abs()
    assert got.shape == y.shape, (what, got.shape, y.shape)
    worst = (err / bound).max().item()
    assert bool((err <= bound).all()), (what, worst)
    return worst
