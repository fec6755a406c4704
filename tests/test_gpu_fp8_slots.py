"""Routed experts in 8 bits, many pairs: the slots' results keep FP32 until their weighted sum has been made, whatever that becomes."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

import fp8_exact as X
from test_gpu_fp8 import check, give, weight
from test_gpu_fp8_experts import by_pair, ids_for

pytestmark = pytest.mark.gpu


def experts_f32(ops, x, g, u, d, wts, ids):
    """The weighted sum in FP32 (C call), with nothing written around its rows."""
    from orin_qwen_lossless_amd import _lib

    T, n_used = ids.shape
    out, L, n = d.rows // d.n_matrices, _lib.lib(), C.c_uint64()
    cg, cu, cd, cx = ops._c_fp8(g), ops._c_fp8(u), ops._c_fp8(d), ops._c_rows("test", x, g.K)
    _lib.check(L.bf16n_fp8_moe_experts_workspace_bytes(C.byref(cg), C.byref(cd), cx.kind, 1, T, n_used, C.byref(n)))
    ws = torch.empty(n.value, dtype=torch.uint8, device="cuda")
    wide = torch.full((T + 2, out), 9.0, device="cuda")
    cy = _lib.Fp8Rows(wide[1:].data_ptr(), None, out * 4, 0, 0, 2, 0)
    _lib.check(L.bf16n_fp8_moe_experts(C.byref(cg), C.byref(cu), C.byref(cd), C.byref(cx), ids.data_ptr(), 0, 4, n_used * 4, wts.data_ptr(), int(wts.dtype is torch.bfloat16), C.byref(cy), T,
                                       n_used, ws.data_ptr(), n.value, ops._stream()))
    assert (wide[0] == 9).all() and (wide[-1] == 9).all()
    return wide[1:-1]


# the last ones: results whose rows are no multiple of eight, few pairs of them among these
@pytest.mark.parametrize("T,n_used,E,mid,K,out", [(60, 4, 8, 144, 256, 256), (300, 2, 4, 96, 1040, 1040), (800, 4, 16, 128, 64, 520), (77, 8, 64, 64, 512, 512), (66, 1, 3, 272, 128, 48), (90, 3, 8, 144, 64, 130),
                                                  (200, 8, 16, 64, 64, 33), (3, 2, 16, 144, 64, 130)])
def test_slots_in_fp32(ops, T, n_used, E, mid, K, out):
    """The layer's own hidden rows, times down in 64 bits, weighted.  A slot's result is off by what FP32 sums are, the weighted sum by a step for each
    slot, and the result by its own rounding: no more, for weights of either sign and sums that nearly cancel."""
    (cg, sg), (cu, su), (cd, sd) = X.matrix(mid, K, 61, E), X.matrix(mid, K, 62, E), X.matrix(out, mid, 63, E)
    g, u, d = weight(ops, cg, sg, E), weight(ops, cu, su, E), weight(ops, cd, sd, E)
    ids = ids_for(T, n_used, E, T + 64)
    dev = ids.to(torch.int32).cuda()
    wts = torch.randn((T, n_used), generator=torch.Generator().manual_seed(65))
    x, _, _ = give(X.rows(T, K, 66, False), "bf16")
    hidden = ops.fp8_moe_mm_ids(x, dev, g, E, u, X.E4M3)
    y, dy = by_pair(hidden.codes.cpu(), hidden.scales.cpu(), cd, sd, ids, E, torch.float32)
    rows = ops.fp8_moe_experts_rows(x, g, u, d, dev, E)
    check(rows.view(T * n_used, out), y, dy)
    for dtype in (torch.float32, torch.bfloat16):
        w = wts.to(dtype)
        y3, d3, w64 = y.view(T, n_used, out), dy.view(T, n_used, out), w.double()[:, :, None]
        total, bound = (y3 * w64).sum(1), (d3 * w64.abs()).sum(1) + (y3 * w64).abs().sum(1) * (n_used + 1) * 2.0 ** -24
        check(ops.fp8_moe_experts(x, g, u, d, w.cuda(), dev, E), total, bound)
        check(experts_f32(ops, x, g, u, d, w.cuda(), dev), total, bound)


def test_as_many_pairs_as_are_by_themselves_and_one_more(ops):
    """Where pairs become lists nothing is lost: the norm of the error stays that of the result's own rounding, 1.66e-3 of that of normal numbers (half a step is
    2^-8 of a power of two; 2^-7 / sqrt(28) of numbers evenly spread from one to the next), within 3 % of it for 2048 of them.  A rounding of each slot
    beside it makes 2.2e-3 and more."""
    E, mid, K, n_used = 64, 512, 256, 8
    (cg, sg), (cu, su), (cd, sd) = X.matrix(mid, K, 71, E), X.matrix(mid, K, 72, E), X.matrix(K, mid, 73, E)
    g, u, d = weight(ops, cg, sg, E), weight(ops, cu, su, E), weight(ops, cd, sd, E)
    for T in (8, 9, 40):
        gen = torch.Generator().manual_seed(74)
        ids = torch.rand((T, E), generator=gen).topk(n_used, 1).indices
        wts = torch.softmax(torch.randn((T, n_used), generator=gen), 1)
        x, _, _ = give(X.rows(T, K, 75, False), "bf16")
        hidden = ops.fp8_moe_mm_ids(x, ids.cuda(), g, E, u, X.E4M3)
        y, _ = by_pair(hidden.codes.cpu(), hidden.scales.cpu(), cd, sd, ids, E, torch.float32)
        total = (y.view(T, n_used, K) * wts.double()[:, :, None]).sum(1)
        got = ops.fp8_moe_experts(x, g, u, d, wts.cuda(), ids.cuda(), E).cpu().double()
        assert (got - total).norm() <= 1.85e-3 * total.norm()


@pytest.mark.parametrize("T,n_used,out", [(70, 8, 520), (300, 3, 64), (90, 2, 33)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_results_at_places_of_any_alignment(ops, T, n_used, out, dtype):
    """The same results wherever they are written (C call), and nothing around them."""
    from orin_qwen_lossless_amd import _lib

    E, mid, K, L, n = 8, 144, 64, _lib.lib(), C.c_uint64()
    g, u, d = weight(ops, *X.matrix(mid, K, 61, E), E), weight(ops, *X.matrix(mid, K, 62, E), E), weight(ops, *X.matrix(out, mid, 63, E), E)
    ids = ids_for(T, n_used, E, 67).to(torch.int32).cuda()
    wts = torch.randn((T, n_used), generator=torch.Generator().manual_seed(68)).cuda()
    x, _, _ = give(X.rows(T, K, 69, False), "bf16")
    cg, cu, cd, cx = ops._c_fp8(g), ops._c_fp8(u), ops._c_fp8(d), ops._c_rows("test", x, K)
    _lib.check(L.bf16n_fp8_moe_experts_workspace_bytes(C.byref(cg), C.byref(cd), cx.kind, 1, T, n_used, C.byref(n)))
    ws = torch.empty(n.value, dtype=torch.uint8, device="cuda")
    want = experts_f32(ops, x, g, u, d, wts, ids).to(dtype)
    assert torch.equal(want, ops.fp8_moe_experts(x, g, u, d, wts, ids, E).to(dtype)) or dtype is torch.float32
    for off in (8, 9, 10, 12):
        y = torch.full((T * out + 24,), 9.0, dtype=dtype, device="cuda")
        cy = _lib.Fp8Rows(y[off:].data_ptr(), None, out * y.element_size(), 0, 0, 1 if dtype is torch.bfloat16 else 2, 0)
        _lib.check(L.bf16n_fp8_moe_experts(C.byref(cg), C.byref(cu), C.byref(cd), C.byref(cx), ids.data_ptr(), 0, 4, n_used * 4, wts.data_ptr(), 0, C.byref(cy), T, n_used, ws.data_ptr(), n.value,
                                           ops._stream()))
        assert torch.equal(y[off: off + T * out].view(T, out), want), off
        assert (y[:off] == 9).all() and (y[off + T * out:] == 9).all(), off
