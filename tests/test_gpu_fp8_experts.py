"""Products in 8 bits by expert, and the routed experts of a layer, against their definition in 64 bits: ragged lists, ids that name no
expert, ids named twice, single tokens."""
from __future__ import annotations

import pytest
import torch

import fp8_exact as X
from test_gpu_fp8 import BF16_HALF, check, give, weight

pytestmark = pytest.mark.gpu


def ids_for(T, n_used, E, seed, odd=True):
    """Ragged: a favoured expert, experts that nothing names, ids that name none, the same one twice."""
    g = torch.Generator().manual_seed(seed)
    p = torch.rand(E, generator=g) ** 3
    ids = torch.multinomial(p + 1e-3, T * n_used, True, generator=g).view(T, n_used)
    if odd and T * n_used > 3:
        ids.view(-1)[1], ids.view(-1)[T * n_used // 2] = -1, E + 3
    return ids


def by_pair(q, xs, c, s, ids, E, out=torch.bfloat16):
    """(y, bound) [pairs, N], zeros where an id names no expert."""
    T, n = ids.shape
    c, s = c.view(E, -1, c.shape[1]), s.view(E, -1, s.shape[1])
    y = torch.zeros((T * n, c.shape[1]), dtype=torch.float64)
    dy = torch.zeros_like(y)
    row = torch.arange(T * n) if q.shape[0] == T * n else torch.arange(T * n) // n
    for e in range(E):
        on = (ids.reshape(-1) == e).nonzero()[:, 0]
        if on.numel():
            y[on], dy[on] = X.product(q[row[on]], xs[row[on]], c[e], s[e], out)
    return y, dy


CASES = [(1, 4, 8, 40, 272), (5, 2, 64, 16, 128), (3, 1, 3, 130, 64), (60, 4, 8, 144, 272), (33, 8, 256, 64, 256), (300, 2, 4, 96, 1040), (500, 1, 2, 256, 512), (200, 8, 64, 176, 128),
         (2, 3, 1, 128, 16), (1000, 4, 16, 32, 64)]


@pytest.mark.parametrize("T,n_used,E,N,K", CASES)
@pytest.mark.parametrize("kind,i64", [("bf16", False), ("rows", True), ("f32", False)])
def test_products_by_expert(ops, T, n_used, E, N, K, kind, i64):
    c, s = X.matrix(N, K, 1, E, kind == "bf16")
    ids = ids_for(T, n_used, E, T)
    dev = ids.to(torch.int64 if i64 else torch.int32).cuda()
    for T_rows in {T, T * n_used}:  # a row to a token, a row to a pair
        x, q, xs = give(X.rows(T_rows, K, 2), kind)
        for out in (torch.float32, torch.bfloat16):
            y, dy = by_pair(q, xs, c, s, ids, E, out)
            got = ops.fp8_moe_mm_ids(x, dev, weight(ops, c, s, E), E, out_dtype=out)
            check(got.view(T * n_used, N), y, dy)
        y, dy = by_pair(q, xs, c, s, ids, E, torch.float32)
        listed = ops.fp8_moe_mm_ids(x, dev, weight(ops, c, s, E), E, routes=ops.int4_route(dev, E))
        check(listed.view(T * n_used, N), y, dy)


@pytest.mark.parametrize("T,n_used,E,N,K", [c for c in CASES if c[3] % 16 == 0])
@pytest.mark.parametrize("kind,out", [("bf16", X.E4M3), ("rows", torch.bfloat16), ("f32", torch.float32), ("rows", X.E4M3)])
def test_gated_by_expert(ops, T, n_used, E, N, K, kind, out):
    (c, s), (cu, su) = X.matrix(N, K, 3, E), X.matrix(N, K, 4, E)
    ids = ids_for(T, n_used, E, T + 1)
    x, q, xs = give(X.rows(T, K, 5, False), kind)
    y, dy = X.gated(*by_pair(q, xs, c, s, ids, E, out), *by_pair(q, xs, cu, su, ids, E, out))
    got = ops.fp8_moe_mm_ids(x, ids.cuda(), weight(ops, c, s, E), E, weight(ops, cu, su, E), out)
    if out is X.E4M3:
        assert X.near_codes(got.codes.cpu(), got.scales.cpu(), y, dy)
    else:
        check(got.view(T * n_used, N), y, dy)


EXPERTS = [(1, 8, 256, 512, 256), (1, 1, 4, 48, 64), (4, 2, 64, 128, 272), (60, 4, 8, 144, 256), (77, 8, 64, 64, 512), (300, 2, 4, 96, 1040), (800, 4, 16, 128, 64), (40, 1, 2, 16, 40 * 16)]


@pytest.mark.parametrize("T,n_used,E,mid,K", EXPERTS)
@pytest.mark.parametrize("kind", ["bf16", "rows"])
def test_experts(ops, T, n_used, E, mid, K, kind):
    """The whole layer against its parts: the hidden rows that the gated product leaves (the layer's own come from the same kernel and are
    rounded to the same codes), times down in 64 bits, weighted."""
    (cg, sg), (cu, su), (cd, sd) = X.matrix(mid, K, 6, E), X.matrix(mid, K, 7, E), X.matrix(K, mid, 8, E)
    g, u, d = weight(ops, cg, sg, E), weight(ops, cu, su, E), weight(ops, cd, sd, E)
    ids = ids_for(T, n_used, E, T + 2)
    dev = ids.to(torch.int32).cuda()
    wts = torch.softmax(torch.randn((T, n_used), generator=torch.Generator().manual_seed(9)), 1)
    x, q, xs = give(X.rows(T, K, 10, False), kind)
    h64, dh = X.gated(*by_pair(q, xs, cg, sg, ids, E), *by_pair(q, xs, cu, su, ids, E))
    hidden = ops.fp8_moe_mm_ids(x, dev, g, E, u, X.E4M3)
    hq, hs = hidden.codes.cpu(), hidden.scales.cpu()
    assert X.near_codes(hq, hs, h64, dh)
    y, dy = by_pair(hq, hs, cd, sd, ids, E)
    rows = ops.fp8_moe_experts_rows(x, g, u, d, dev, E)
    check(rows.view(T * n_used, K), y, dy)
    dy = dy + (y.abs() + dy) * BF16_HALF  # the slots' results may be held in BF16
    y3, d3 = y.view(T, n_used, K), dy.view(T, n_used, K)
    for dtype in (torch.float32, torch.bfloat16):
        wt = wts.to(dtype)
        w = wt.double()[:, :, None]
        total, bound = (y3 * w).sum(1), (d3 * w).sum(1) + (y3 * w).abs().sum(1) * (n_used + 1) * 2.0 ** -24
        got = ops.fp8_moe_experts(x, g, u, d, wt.cuda(), dev, E)
        assert got.dtype is torch.bfloat16
        check(got, total, bound)


def test_nothing_named(ops):
    E, mid, K = 4, 32, 64
    g, u, d = (weight(ops, *X.matrix(*sh, 1, E), E) for sh in ((mid, K), (mid, K), (K, mid)))
    for T in (1, 40):
        x = torch.randn((T, K), device="cuda").to(torch.bfloat16)
        ids = torch.full((T, 3), -7, dtype=torch.int64, device="cuda")
        ids[:, 1] = 1 << 33  # (the low word names one)
        assert not ops.fp8_moe_experts(x, g, u, d, torch.ones((T, 3), device="cuda"), ids, E).any()
        h = ops.fp8_moe_mm_ids(x, ids, g, E, u, X.E4M3)
        assert not h.codes.float().any() and (h.scales == 2.0 ** -100 / 448).all()
    assert ops.fp8_moe_experts(x[:0], g, u, d, torch.ones((0, 3), device="cuda"), ids[:0], E).shape == (0, K)
    assert ops.fp8_moe_experts_rows(x[:0], g, u, d, ids[:0], E).shape == (0, 3, K)


def test_wider_rows_of_ids(ops):
    E, mid, K, T = 4, 32, 64, 30
    g, u, d = (weight(ops, *X.matrix(*sh, 1, E), E) for sh in ((mid, K), (mid, K), (K, mid)))
    x = torch.randn((T, K), device="cuda").to(torch.bfloat16)
    wide = torch.randint(0, E, (T, 9), dtype=torch.int32, device="cuda")
    w = torch.rand((T, 2), device="cuda")
    for n in (1, T):
        assert torch.equal(ops.fp8_moe_experts(x[:n], g, u, d, w[:n], wide[:n, 3:5], E), ops.fp8_moe_experts(x[:n], g, u, d, w[:n], wide[:n, 3:5].contiguous(), E))


def test_refusals(ops):
    E, mid, K, T = 4, 32, 64, 3
    g, u, d = (weight(ops, *X.matrix(*sh, 1, E), E) for sh in ((mid, K), (mid, K), (K, mid)))
    x, ids, w = torch.zeros((T, K), dtype=torch.bfloat16, device="cuda"), torch.zeros((T, 2), dtype=torch.int32, device="cuda"), torch.ones((T, 2), device="cuda")
    for call in (lambda: ops.fp8_moe_experts(x, g, u, d, w, ids, 5), lambda: ops.fp8_moe_experts(x, g, u, g, w, ids, E), lambda: ops.fp8_moe_experts(x, g, d, d, w, ids, E),
                 lambda: ops.fp8_moe_experts(x, g, u, d, w[:, :1], ids, E), lambda: ops.fp8_moe_experts(x, g, u, d, None, ids, E), lambda: ops.fp8_moe_experts(x[:2], g, u, d, w, ids, E),
                 lambda: ops.fp8_moe_experts(x, g, u, d, w, ids.float(), E), lambda: ops.fp8_moe_experts(x, g, u, d, w, ids.cpu(), E), lambda: ops.fp8_moe_mm_ids(x, ids, g, E, out_dtype=X.E4M3),
                 lambda: ops.fp8_moe_mm_ids(x[:2], ids, g, E), lambda: ops.fp8_moe_mm_ids(x, ids, g, E, d), lambda: ops.fp8_moe_mm_ids(x, ids, g, E, routes=ops.int4_route(ids[:2], E)),
                 lambda: ops.fp8_moe_mm_ids(x.half(), ids, g, E), lambda: ops.fp8_moe_experts(x, g, u, d, w.half(), ids, E)):
        with pytest.raises(ValueError):
            call()
