"""The norm in 8 bits of addends that lie far apart: their sum is held in 64 bits, as the squares' is."""
from __future__ import annotations

import pytest
import torch

import fp8_exact as X

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,n,slots", [(1, 64, 0), (5, 2048, 0), (40, 272, 0), (3, 16384, 0), (5, 2576, 3), (2, 16384, 9), (2, 9008, 5)])
@pytest.mark.parametrize("given", ["ab", "abc"])
def test_addends_far_apart(ops, T, n, slots, given):
    """a and c cancel but for b, which is 2^-12 to 2^-30 of them: FP32 loses most or all of b's bits.  Sums of so few numbers of 8 bits are exact in 64,
    a slot's product of 24 bits and 24 too, so that rows, scales and the BF16 sum are the definition's own (an element of 64-bit arithmetic that falls on the
    other side of the middle of two FP32 numbers, and that of two codes: 2^-53 against 2^-24, one in 2^29 of them at most)."""
    g = torch.Generator().manual_seed(T * n + slots)
    r = lambda *sh: torch.randn(sh, generator=g)  # noqa: E731
    a = (r(T, n) * 2.0 ** 10).to(torch.bfloat16)
    b = (r(T, n) * torch.exp2(-torch.randint(2, 21, (T, n), generator=g).float())).to(torch.bfloat16)
    c = -a if given == "abc" else None
    gamma = (1 + 0.3 * r(n)).to(torch.bfloat16)
    ys, wts = (r(T, slots, n) * 2.0 ** -10, torch.softmax(r(T, slots), 1)) if slots else (None, None)
    s = a.double() + b.double() + (0 if c is None else c.double())
    for k in range(slots):
        s = s + wts[:, k, None].double() * ys[:, k].double()
    eps = torch.tensor(1e-6, dtype=torch.float32).double()
    y = (s / torch.sqrt(s.square().mean(1, keepdim=True) + eps) * gamma.double()).float()
    d = lambda t: None if t is None else t.cuda()  # noqa: E731
    rows, total, norm = ops.add_rmsnorm_fp8(d(a), d(b), d(c), d(ys), d(wts), d(gamma), want_sum=True, want_norm=True)
    q, qs = X.quantize(y)
    assert torch.equal(total.cpu(), s.float().to(torch.bfloat16))
    assert torch.equal(norm.cpu(), y.to(torch.bfloat16))
    assert torch.equal(rows.codes.cpu().view(torch.uint8), q.view(torch.uint8)) and torch.equal(rows.scales.cpu(), qs)
