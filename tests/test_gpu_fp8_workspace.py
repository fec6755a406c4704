"""8-bit floating point with block scales: one workspace, sized once for the longest batch, serves every shorter one."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

import fp8_exact as X
from test_gpu_fp8 import give, weight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["bf16", "rows"])
def test_gated_products_of_every_count(ops, kind):
    from orin_qwen_lossless_amd import _lib

    R, K, most, L, n = 1408, 1040, 120, _lib.lib(), C.c_uint64()
    g, u = (weight(ops, *X.matrix(R, K, 91 + i)) for i in range(2))
    cg, cu = ops._c_fp8(g), ops._c_fp8(u)
    x, q, xs = give(X.rows(most, K, 93, False), kind)
    kinds = ops._c_rows("test", x, K).kind
    _lib.check(L.bf16n_fp8_workspace_bytes(C.byref(cg), 1, kinds, 0, most, 0, 0, C.byref(n)))
    ws = torch.empty(n.value, dtype=torch.uint8, device="cuda")
    for T in (most, 100, 94, 93, 88, 64, 17, 16, 1):
        rows = ops.Fp8Rows(x.codes[:T], x.scales[:T]) if kind == "rows" else x[:T]
        y, cy = ops._fp8_out(T, R, X.E4M3, torch.device("cuda"))
        cx = ops._c_rows("test", rows, K)
        _lib.check(L.bf16n_fp8_mm(C.byref(cg), C.byref(cu), C.byref(cx), C.byref(cy), T, ws.data_ptr(), n.value, ops._stream()))
        want = ops.fp8_linear_glu2(rows, g, u, X.E4M3)
        assert torch.equal(y.codes.view(torch.uint8), want.codes.view(torch.uint8)) and torch.equal(y.scales, want.scales)


@pytest.mark.parametrize("kind", ["bf16", "rows"])
def test_experts_of_every_count(ops, kind):
    from orin_qwen_lossless_amd import _lib

    E, mid, K, n_used, most, L, n = 64, 144, 64, 4, 18, _lib.lib(), C.c_uint64()
    g, u, d = weight(ops, *X.matrix(mid, K, 94, E), E), weight(ops, *X.matrix(mid, K, 95, E), E), weight(ops, *X.matrix(K, mid, 96, E), E)
    cg, cu, cd = (ops._c_fp8(w) for w in (g, u, d))
    x, _, _ = give(X.rows(most, K, 97, False), kind)
    ids = torch.randint(0, E, (most, n_used), generator=torch.Generator().manual_seed(98), dtype=torch.int32).cuda()
    wts = torch.rand((most, n_used), generator=torch.Generator().manual_seed(99)).cuda()
    _lib.check(L.bf16n_fp8_moe_experts_workspace_bytes(C.byref(cg), C.byref(cd), ops._c_rows("test", x, K).kind, 0, most, n_used, C.byref(n)))
    ws = torch.empty(n.value, dtype=torch.uint8, device="cuda")
    for T in (most, 17, 16, 15, 1):  # (16 tokens' pairs are as many as are products by themselves)
        rows = ops.Fp8Rows(x.codes[:T], x.scales[:T]) if kind == "rows" else x[:T]
        y, cy = ops._fp8_out(T * n_used, K, torch.float32, torch.device("cuda"))
        cx = ops._c_rows("test", rows, K)
        _lib.check(L.bf16n_fp8_moe_experts(C.byref(cg), C.byref(cu), C.byref(cd), C.byref(cx), ids.data_ptr(), 0, 4, n_used * 4, None, 0, C.byref(cy), T, n_used, ws.data_ptr(), n.value, ops._stream()))
        assert torch.equal(y.view(T, n_used, K), ops.fp8_moe_experts_rows(rows, g, u, d, ids[:T], E))
