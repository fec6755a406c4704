"""8-bit floating point with block scales in 64 bits: values of rows and matrices, their products, and how far FP32 sums may be off."""
from __future__ import annotations

import torch

BLOCK = 128
E4M3 = torch.float8_e4m3fn


def spread(s: torch.Tensor, K: int) -> torch.Tensor:
    return s.double().repeat_interleave(BLOCK, 1)[:, :K]


def quantize(v: torch.Tensor):
    """(codes, scales) of FP32 rows on the CPU: IEEE quotients and product, torch's rounding to nearest even."""
    v = v.float()
    T, K = v.shape
    b = torch.nn.functional.pad(v, (0, -K % BLOCK)).view(T, -1, BLOCK)
    m = torch.where(b.isnan(), 0.0, b.abs()).amax(2).clamp_min(2.0 ** -100)
    q = (b * (torch.full_like(m, 448.0) / m)[:, :, None]).to(E4M3)  # (448.0 / m would be a product with a reciprocal)
    return q.view(T, -1)[:, :K].contiguous(), m / 448.0


def rows(T, K, seed, wide=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((T, K), generator=g)
    return x * torch.exp2(torch.randint(-6, 7, (T, K), generator=g).float()) if wide else x


def matrix(rows_, K, seed, n=1, bf16=False):
    """codes over all of e4m3's finite values, scales [n * blocks of rows, blocks of columns]"""
    g = torch.Generator().manual_seed(seed)
    codes = (torch.randn((n * rows_, K), generator=g) * 100).clamp_(-448, 448)
    codes = torch.where(torch.rand((n * rows_, K), generator=g) < 0.1, codes * 2.0 ** -12, codes).to(E4M3)
    scales = (0.5 + torch.rand((n * -(-rows_ // BLOCK), -(-K // BLOCK)), generator=g)) * 2e-4
    return codes, scales.to(torch.bfloat16) if bf16 else scales


def weight64(codes, scales, n=1):
    """[n, rows, K]"""
    R, K = codes.shape[0] // n, codes.shape[1]
    s = scales.double().view(n, -1, scales.shape[1])
    return codes.double().view(n, R, K) * s.repeat_interleave(BLOCK, 1)[:, :R].repeat_interleave(BLOCK, 2)[:, :, :K]


def product(xq, xs, c, s, out=torch.float32):
    """(y, bound on its error) of rows in codes and one matrix, codes c and scales s, in 64 bits.  Up to 128 terms are added within the matrix cores, where
    a step may be lost at each (2^-23), then come a product of scales, one fmaf to a block and up to eight parts' sums (2^-24 each).
    Results that are not FP32 may come from the instruction on the codes: of eight consecutive columns' products it drops what is below
    2^-13 of the largest one, by exponents (numbers below 2^-6 have that one's): seven times at most."""
    K = xq.shape[1]
    x, w = xq.double() * spread(xs, K), weight64(c, s)[0]
    size = x.abs() @ w.abs().t()
    bound = size * (128 * 2.0 ** -23 + (-(-K // BLOCK) + 10) * 2.0 ** -24) + 2.0 ** -140
    if out is not torch.float32:
        most = lambda q, scales: (q.double().abs().clamp_min(2.0 ** -6) * scales).view(q.shape[0], K // 8, 8).amax(2)  # noqa: E731
        rows_ = s.double().repeat_interleave(BLOCK, 0)[: c.shape[0]].repeat_interleave(BLOCK, 1)[:, :K]
        bound = bound + 7 * 2.0 ** -13 * (most(xq, spread(xs, K)) @ most(c, rows_).t())
    return x @ w.t(), bound


def gated(g, dg, u, du):
    """silu(g) * u and its bound: |silu'| <= 1.1, an exponential off by a few steps (2^-20 of the value)."""
    y = g * torch.sigmoid(g) * u
    return y, 1.1 * dg * (u.abs() + du) + (g * torch.sigmoid(g)).abs() * du + y.abs() * 2.0 ** -20 + 2.0 ** -126


def near_codes(got_q, got_s, y, dy):
    """Whether codes with scales are a rounding of y, which the kernel had within dy."""
    T, K = y.shape
    pad = lambda t: torch.nn.functional.pad(t, (0, -K % BLOCK)).view(T, -1, BLOCK)  # noqa: E731
    most, off = pad(y.abs()).amax(2).clamp_min(2.0 ** -100), pad(dy).amax(2)
    assert ((got_s.double() - most / 448).abs() <= off / 448 + most / 448 * 2.0 ** -23).all()
    v = got_q.double() * spread(got_s, K)
    step = torch.maximum(y.abs() * 2.0 ** -4, spread(got_s, K) * 2.0 ** -10)  # half a step of e4m3; half of its smallest number
    return ((v - y).abs() <= step * (1 + 2.0 ** -20) + dy * 1.07).all()
