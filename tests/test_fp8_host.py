"""8-bit floating point with block scales, without a GPU: what the classes and the calls refuse, the quantization of weights."""
from __future__ import annotations

import pytest
import torch

import fp8_exact as X
from orin_qwen_lossless_amd import _lib, ops


def test_the_weights_class_refuses_what_the_kernels_do_not_take():
    c, s = X.matrix(150, 144, 1, 2)
    w = ops.Fp8Weight(c, s, 2)
    assert (w.rows, w.K, w.nbytes) == (300, 144, c.numel() + 4 * s.numel()) and w.to("cpu").n_matrices == 2
    assert ops.Fp8Weight(c, s[:3].contiguous(), 1).n_matrices == 1  # (300 rows are three blocks; twice 150 are four)
    for bad in ((c.view(torch.uint8), s, 2), (c.view(torch.float8_e5m2), s, 2), (c[:, ::2], s, 2), (c.reshape(-1), s, 2), (c[:, :40].contiguous(), s, 2), (c, s.half(), 2), (c, s[:3], 2),
                (c, s, 1), (c, s, 7), (c, s, 0), (c, s, 2.0), (c, s, True), (c, s[:, :1].contiguous(), 2), (c, s.t().contiguous().t(), 2),
                (torch.zeros((1, 32784)).to(X.E4M3), torch.ones((1, 257)), 1)):
        with pytest.raises(ValueError):
            ops.Fp8Weight(*bad)


def test_the_rows_class():
    q, s = X.quantize(X.rows(5, 272, 1))
    r = ops.Fp8Rows(q, s)
    assert torch.equal(r.dequant().double(), (q.float() * X.spread(s, 272).float()).double())
    ops.Fp8Rows(q, s.t().contiguous().t())
    for bad in ((q.float(), s), (q, s[:4]), (q, s[:, :2]), (q, s.double()), (q.t(), s), (q[0], s[0])):
        with pytest.raises(ValueError):
            ops.Fp8Rows(*bad)


def test_calls_refuse_host_tensors():
    w = ops.Fp8Weight(*X.matrix(64, 64, 1))
    x, ids, one = torch.zeros((2, 64), dtype=torch.bfloat16), torch.zeros((2, 1), dtype=torch.int32), torch.ones((2, 1))
    rows = ops.Fp8Rows(*X.quantize(x))
    for call in (lambda: ops.fp8_linear(x, w), lambda: ops.fp8_linear(rows, w), lambda: ops.fp8_linear_glu2(x, w, w), lambda: ops.fp8_quantize_rows(x), lambda: ops.add_rmsnorm_fp8(x),
                 lambda: ops.fp8_moe_mm_ids(x, ids, w, 1), lambda: ops.fp8_moe_experts(x, w, w, w, one, ids, 1), lambda: ops.fp8_moe_experts_rows(x, w, w, w, ids, 1)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("shape,n", [((300, 272), 1), ((4, 70, 48), 4), ((1, 16), 1), ((256, 128), 2)])
@pytest.mark.parametrize("scale_dtype", [torch.float32, torch.bfloat16])
def test_quantize(shape, n, scale_dtype, monkeypatch):
    monkeypatch.setattr(ops, "DEQUANT_CHUNK_BYTES", 1 << 16)  # (pieces of one block of rows)
    w = torch.randn(shape, generator=torch.Generator().manual_seed(1)) * 0.02
    w.view(-1, shape[-1])[:, :16] *= 100
    w.view(-1, shape[-1])[0] = 0
    q = ops.fp8_quantize(w, n, scale_dtype)
    v = X.weight64(q.codes, q.scales, n).view(-1, shape[-1])
    s = X.weight64(torch.ones(q.codes.shape).to(X.E4M3), q.scales, n).view(-1, shape[-1])
    x = w.view(-1, shape[-1]).double()
    # half a step; a scale in BF16 may be half of its step too small, the largest code standing for that much less
    assert ((v - x).abs() <= torch.maximum(x.abs() * (2.0 ** -4 + 2.0 ** -20), s * 2.0 ** -10)).all()
    assert not v[0].any() and torch.isfinite(q.codes.float()).all()


def test_quantize_of_special_weights():
    w = torch.randn((256, 256), generator=torch.Generator().manual_seed(2))
    w[3, 5], w[200, 7] = float("nan"), float("inf")
    q = ops.fp8_quantize(w)
    v = X.weight64(q.codes, q.scales)[0]
    assert v[:, 128:].isfinite().all() and not v[3, 5].isfinite() and not v[200, 7].isfinite()
    assert (ops.fp8_quantize(torch.zeros((16, 16))).scales > 0).all()
    for bad in (lambda: ops.fp8_quantize(w[0]), lambda: ops.fp8_quantize(w[:, :40]), lambda: ops.fp8_quantize(w.half()), lambda: ops.fp8_quantize(w, 3), lambda: ops.fp8_quantize(w, 0),
                lambda: ops.fp8_quantize(w, scale_dtype=torch.float16)):
        with pytest.raises(ValueError):
            bad()


def test_workspace_sizes_and_refusals_of_the_c_calls():
    """Without a device: sizes are computed, wrong descriptions refused, both with a message."""
    import ctypes as C

    L, n = _lib.lib(), C.c_uint64()
    w = _lib.Fp8Weight(4096, 4096, 256, 512, 4, 0, 0)
    ask = lambda w, **k: L.bf16n_fp8_workspace_bytes(C.byref(w), k.get("up", 0), k.get("x", 1), k.get("y", 1), k.get("rows", 100), k.get("pairs", 0), 1, C.byref(n))  # noqa: E731
    assert ask(w) == 0 and n.value >= 100 * 256 + 100 * 2 * 4  # BF16 rows of many tokens become codes
    assert ask(w, x=0) == 0 and n.value == 0
    assert ask(w, x=0, y=0, up=1, rows=3) == 0 and n.value >= 3 * 128 * 4
    for field, value in (("K", 40), ("K", 0), ("K", 32784), ("n_matrices", 0), ("n_matrices", 3), ("n_matrices", 65535), ("codes", 4100), ("scales", 4098), ("codes", None), ("rows", -4),
                         ("rows", 1 << 40)):
        bad = _lib.Fp8Weight(4096, 4096, 256, 512, 4, 0, 0)
        setattr(bad, field, value)
        assert ask(bad) == _lib.EINVAL and L.bf16n_last_error().startswith(b"bf16n: fp8")
    assert ask(w, rows=-1) == _lib.EINVAL
    down = _lib.Fp8Weight(4096, 4096, 128, 1024, 4, 0, 0)
    assert L.bf16n_fp8_moe_experts_workspace_bytes(C.byref(w), C.byref(down), 1, 1, 10, 2, C.byref(n)) == 0 and n.value > 20 * 128
    for args in ((0, 2), (10, 0), (65536, 2), (10, 1024)):
        assert L.bf16n_fp8_moe_experts_workspace_bytes(C.byref(w), C.byref(down), 1, 1, *args, C.byref(n)) == _lib.EINVAL
    assert L.bf16n_fp8_moe_experts_workspace_bytes(C.byref(w), C.byref(w), 1, 1, 10, 2, C.byref(n)) == _lib.EINVAL
