"""8-bit floating point with a scale for every block of 128 against its definition in 64 bits: rows, the norm, dense and gated products."""
from __future__ import annotations

import pytest
import torch

import fp8_exact as X

pytestmark = pytest.mark.gpu
BF16_HALF = torch.finfo(torch.bfloat16).eps / 2


def give(x, kind):
    """Rows [T, K] on the CPU as (what the call gets, codes, scales on the CPU)."""
    from orin_qwen_lossless_amd import ops

    x = x.to(torch.bfloat16) if kind == "bf16" else x
    q, s = X.quantize(x)
    return (ops.Fp8Rows(q.cuda(), s.cuda()) if kind == "rows" else x.cuda()), q, s


def weight(ops, c, s, n=1):
    return ops.Fp8Weight(c.cuda(), s.cuda(), n)


def check(got, y, dy):
    assert got.shape == y.shape
    if got.dtype is torch.bfloat16:
        dy = dy + (y.abs() + dy) * BF16_HALF
    assert ((got.cpu().double() - y).abs() <= dy).all()


@pytest.mark.parametrize("T,K", [(1, 16), (3, 128), (5, 2576), (7, 272), (2, 32768), (300, 96)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_bit_for_bit(ops, T, K, dtype):
    x = X.rows(T, K, T + K).to(dtype)
    x[0, : min(K, 40)] = 0
    if T > 2:
        x[1], x[2] = 0, x[2] * 1e-36
    q, s = X.quantize(x)
    r = ops.fp8_quantize_rows(x.cuda())
    assert torch.equal(r.codes.cpu().view(torch.uint8), q.view(torch.uint8)) and torch.equal(r.scales.cpu(), s)
    wide = torch.randn((T, K + 32)).to(dtype)
    wide[:, 16: 16 + K] = x
    r = ops.fp8_quantize_rows(wide.cuda()[:, 16: 16 + K])
    assert torch.equal(r.codes.cpu().view(torch.uint8), q.view(torch.uint8)) and torch.equal(r.scales.cpu(), s)
    assert (r.dequant().cpu() - q.float() * X.spread(s, K).float()).abs().max() == 0


def test_rows_of_special_values(ops):
    """The largest numbers, ties, denormals, NaN and infinities: a block with an infinity has an infinite scale, others do not notice."""
    x = X.rows(6, 256, 3)
    x[0] = torch.finfo(torch.float32).max
    x[1, :128], x[1, 5] = torch.linspace(-448, 448, 128), 448.0  # (scale 1: ties between codes among them)
    x[2] = 2.0 ** -140
    x[3, 7], x[4, 9], x[5, 200] = float("nan"), float("inf"), -float("inf")
    q, s = X.quantize(x)
    r = ops.fp8_quantize_rows(x.cuda())
    got, want = r.codes.cpu(), q
    assert torch.equal(r.scales.cpu(), s) and s[4, 0] == float("inf") and s[4, 1] < 1 and s[3].isfinite().all()
    nan = want.float().isnan()
    assert torch.equal(got.float().isnan(), nan) and nan.sum() == 3
    assert torch.equal(got.view(torch.uint8)[~nan], want.view(torch.uint8)[~nan])


SHAPES = [(1, 16, 1), (17, 128, 3), (130, 272, 16), (512, 2048, 1), (300, 1040, 33), (257, 512, 100), (1453, 2576, 19), (129, 144, 200), (16, 32768, 2),
          (128, 4096, 17), (700, 2048, 500), (40, 640, 1000), (3000, 256, 8), (20000, 512, 5)]


@pytest.mark.parametrize("R,K,T", SHAPES)
@pytest.mark.parametrize("kind,bf16_scales,out", [("bf16", False, torch.bfloat16), ("f32", True, torch.float32), ("rows", False, torch.float32)])
def test_linear(ops, R, K, T, kind, bf16_scales, out):
    c, s = X.matrix(R, K, R + K, bf16=bf16_scales)
    x, q, xs = give(X.rows(T, K, T), kind)
    y, dy = X.product(q, xs, c, s, out)
    check(ops.fp8_linear(x, weight(ops, c, s), out_dtype=out), y, dy)


@pytest.mark.parametrize("R,K,T", [(16, 16, 1), (48, 272, 3), (144, 512, 16), (512, 2048, 1), (1408, 1040, 33), (272, 256, 300), (128, 128, 64), (64, 16384, 9), (256, 2048, 129)])
@pytest.mark.parametrize("kind,out", [("bf16", torch.bfloat16), ("f32", X.E4M3), ("rows", X.E4M3), ("rows", torch.float32)])
def test_gated(ops, R, K, T, kind, out):
    (c, s), (cu, su) = X.matrix(R, K, R), X.matrix(R, K, R + 1)
    x, q, xs = give(X.rows(T, K, T, False), kind)
    y, dy = X.gated(*X.product(q, xs, c, s, out), *X.product(q, xs, cu, su, out))
    got = ops.fp8_linear_glu2(x, weight(ops, c, s), weight(ops, cu, su), out_dtype=out)
    if out is X.E4M3:
        assert got.codes.shape == (T, R) and X.near_codes(got.codes.cpu(), got.scales.cpu(), y, dy)
    else:
        check(got, y, dy)


@pytest.mark.parametrize("T", [1, 20, 70])
def test_bias_leading_axes_and_strides(ops, T):
    R, K = 200, 256
    c, s = X.matrix(R, K, 1)
    w = weight(ops, c, s)
    bias = torch.randn(R, generator=torch.Generator().manual_seed(2))
    x, q, xs = give(X.rows(2 * T, K, 3), "bf16")
    y, dy = X.product(q, xs, c, s)
    check(ops.fp8_linear(x.view(2, T, K), w, bias.cuda()).view(2 * T, R), y + bias, dy + (y + bias).abs() * 2.0 ** -24 + 2.0 ** -24 * dy)
    odd = torch.empty((2 * T, K + 3), dtype=torch.bfloat16, device="cuda")
    odd[:, 1: K + 1] = x
    assert torch.equal(ops.fp8_linear(odd[:, 1: K + 1], w), ops.fp8_linear(x, w))  # (copied to aligned rows first)
    wide = torch.zeros((2 * T, K + 64), dtype=torch.bfloat16, device="cuda")
    wide[:, 32: K + 32] = x
    assert torch.equal(ops.fp8_linear(wide[:, 32: K + 32], w), ops.fp8_linear(x, w))
    # codes in wider rows, their scales by rows instead of by blocks
    wc = torch.zeros((2 * T, K + 32), dtype=torch.uint8, device="cuda").view(X.E4M3)
    wc.view(torch.uint8)[:, 16: K + 16] = q.cuda().view(torch.uint8)
    r = ops.Fp8Rows(wc[:, 16: K + 16], xs.cuda().contiguous())
    assert torch.equal(ops.fp8_linear(r, w), ops.fp8_linear(x, w)) and torch.equal(ops.fp8_linear(r, w), ops.fp8_linear(ops.fp8_quantize_rows(x), w))


@pytest.mark.parametrize("T", [1, 16, 17, 100])
def test_values_that_are_not_finite(ops, T):
    """An activation that is not finite makes its row NaN, a weight its column; nothing else notices (the next row's first columns, which
    stand where a cut block's chunks would be, among it)."""
    R, K = 150, 272
    c, s = X.matrix(R, K, 4)
    c.view(torch.uint8)[149] = 0x7F
    c.view(torch.uint8)[3, 271] = 0xFF
    x = X.rows(T, K, 5)
    bad = [0] if T == 1 else [0, T - 1]
    x[0, 17] = float("inf")
    x[bad[-1], 260] = float("nan")
    for kind in ("bf16", "rows"):
        given, q, xs = give(x, kind)
        got = ops.fp8_linear(given, weight(ops, c, s), out_dtype=torch.float32).cpu()
        nan = torch.zeros((T, R), dtype=torch.bool)
        nan[:, 149] = nan[:, 3] = True
        nan[bad] = True
        assert torch.equal(got.isnan(), nan)
        y, dy = X.product(torch.where(q.float().isnan(), 0.0, q.float()), torch.where(xs.isinf(), 1.0, xs), torch.nan_to_num(c.float(), nan=0.0), s)
        assert ((got.double() - y).abs() <= dy)[~nan].all()


def test_nothing_behind_the_results(ops):
    """The rows around a result stay as they were (C call)."""
    import ctypes as C

    from orin_qwen_lossless_amd import _lib

    for R, K, T in ((130, 272, 19), (130, 272, 200), (1, 16, 40)):
        c, s = X.matrix(R, K, 6)
        w = weight(ops, c, s)
        x, q, xs = give(X.rows(T, K, 7), "rows")
        y, dy = X.product(q, xs, c, s)
        wide = torch.full((T + 2, R + 5), 9.0, device="cuda")
        cw, cx = ops._c_fp8(w), ops._c_rows("test", x, K)
        cy = _lib.Fp8Rows(wide[1:, 3:].data_ptr(), None, wide.stride(0) * 4, 0, 0, 2, 0)
        _lib.check(_lib.lib().bf16n_fp8_mm(C.byref(cw), None, C.byref(cx), C.byref(cy), T, None, 0, ops._stream()))
        check(wide[1: T + 1, 3: R + 3], y, dy)
        wide[1: T + 1, 3: R + 3] = 9
        assert (wide == 9).all()


@pytest.mark.parametrize("T,n,slots", [(1, 2048, 0), (5, 16, 0), (3, 272, 2), (333, 2576, 8), (2, 16384, 1), (40, 4096, 0), (700, 2048, 9), (9, 6000, 3), (4, 1024, 40)])
def test_norm(ops, T, n, slots):
    g = torch.Generator().manual_seed(T + n)
    r = lambda *sh: torch.randn(sh, generator=g)  # noqa: E731
    a, b, c = ((r(T, n) * k).to(torch.bfloat16) for k in (3, 1, 0.1))
    gamma = (1 + 0.3 * r(n)).to(torch.bfloat16)
    ys, wts = (r(T, slots, n), torch.softmax(r(T, slots), 1)) if slots else (None, None)
    if T > 2:
        a[1] = b[1] = c[1] = 0  # a row of zeros
        if slots:
            ys[1] = 0
    d = lambda t: None if t is None else t.cuda()  # noqa: E731
    got, total, norm = ops.add_rmsnorm_fp8(d(a), d(b), d(c), d(ys), d(wts), d(gamma), 1e-6, True, True)
    s = a.double() + b.double() + c.double()
    size = a.double().abs() + b.double().abs() + c.double().abs()
    if slots:
        s, size = s + (ys.double() * wts.double()[:, :, None]).sum(1), size + (ys.double() * wts.double()[:, :, None]).abs().sum(1)
    ds = size * (slots + 3) * 2.0 ** -24
    inv = 1 / torch.sqrt(s.square().mean(1, keepdim=True) + 1e-6)
    # the mean of squares: off by twice the terms' relative errors, and by n roundings of a sum of positive numbers
    rel = (2 * (s.abs() * ds).sum(1, keepdim=True) / s.square().sum(1, keepdim=True).clamp_min(1e-30) + (n / 256 + 16) * 2.0 ** -24) / 2 + 4 * 2.0 ** -24
    y = s * inv * gamma.double()
    dy = (ds * inv * gamma.double().abs()) + y.abs() * (rel + 2 * 2.0 ** -24)
    assert X.near_codes(got.codes.cpu(), got.scales.cpu(), y, dy)
    check(total, s, ds)
    check(norm, y, dy)
    alone = ops.add_rmsnorm_fp8(d(a), d(b), d(c), d(ys), d(wts), d(gamma))
    assert torch.equal(alone.codes.view(torch.uint8), got.codes.view(torch.uint8)) and torch.equal(alone.scales, got.scales)
    # no gamma, BF16 weights
    if slots:
        w16 = wts.to(torch.bfloat16)
        r16, t16 = ops.add_rmsnorm_fp8(d(a), ys=d(ys), topk_weights=d(w16), want_sum=True)
        s16 = a.double() + (ys.double() * w16.double()[:, :, None]).sum(1)
        check(t16, s16, ds + (ys.double() * w16.double()[:, :, None]).abs().sum(1) * (slots + 3) * 2.0 ** -24)
    else:
        assert torch.equal(ops.add_rmsnorm_fp8(d(a), want_norm=True)[1], ops.add_rmsnorm_fp8(d(a), gamma=torch.ones(n, dtype=torch.bfloat16, device="cuda"), want_norm=True)[1])


def test_norm_of_values_that_are_not_finite(ops):
    a = X.rows(3, 512, 1, False).to(torch.bfloat16)
    a[0, 3], a[1, 400] = float("nan"), float("inf")
    r = ops.add_rmsnorm_fp8(a.cuda())
    assert r.codes.cpu().float()[0].isnan().all() and r.codes.cpu().float()[1, 400].isnan()
    assert r.codes.cpu().float()[2].isfinite().all() and r.scales[2].isfinite().all()


def test_nothing_to_do(ops):
    c, s = X.matrix(40, 64, 1)
    w = weight(ops, c, s)
    for dtype in (torch.bfloat16, torch.float32):
        none = torch.empty((0, 64), dtype=dtype, device="cuda")
        assert ops.fp8_linear(none, w).shape == (0, 40) and ops.fp8_quantize_rows(none).codes.shape == (0, 64)
        assert ops.fp8_linear_glu2(ops.fp8_quantize_rows(none), w, w, torch.float32).shape == (0, 40)
    assert ops.add_rmsnorm_fp8(torch.empty((0, 64), dtype=torch.bfloat16, device="cuda"), want_sum=True)[1].shape == (0, 64)
    empty = ops.Fp8Weight(w.codes[:0], w.scales[:0], 1)
    assert ops.fp8_linear(torch.zeros((3, 64), dtype=torch.bfloat16, device="cuda"), empty).shape == (3, 0)


def test_refusals(ops):
    c, s = X.matrix(40, 64, 1)
    w = weight(ops, c, s)
    x = torch.zeros((2, 64), dtype=torch.bfloat16, device="cuda")
    stack = ops.Fp8Weight(w.codes, torch.ones((4, 1), device="cuda"), 4)
    for call in (lambda: ops.fp8_linear(x.half(), w), lambda: ops.fp8_linear(x[:, :48], w), lambda: ops.fp8_linear(x.cpu(), w), lambda: ops.fp8_linear(x, w, out_dtype=X.E4M3),
                 lambda: ops.fp8_linear(x, stack), lambda: ops.fp8_linear_glu2(x, w, weight(ops, *X.matrix(41, 64, 1))), lambda: ops.fp8_linear_glu2(x, w, w, X.E4M3),
                 lambda: ops.fp8_linear_glu2(x, w, w, torch.float16), lambda: ops.fp8_linear(x[:, 4:], w), lambda: ops.fp8_quantize_rows(x[:, :40]), lambda: ops.fp8_quantize_rows(x[0]),
                 lambda: ops.fp8_quantize_rows(x.half()), lambda: ops.add_rmsnorm_fp8(x[:, :40].contiguous()), lambda: ops.add_rmsnorm_fp8(x.float()),
                 lambda: ops.add_rmsnorm_fp8(x, x[:1]), lambda: ops.add_rmsnorm_fp8(x, gamma=x[0].float()), lambda: ops.add_rmsnorm_fp8(x, ys=torch.zeros((2, 1, 64), device="cuda")),
                 lambda: ops.add_rmsnorm_fp8(torch.zeros((1, 16400), dtype=torch.bfloat16, device="cuda")), lambda: ops.add_rmsnorm_fp8(x, gamma=x[0].cpu())):
        with pytest.raises(ValueError):
            call()
