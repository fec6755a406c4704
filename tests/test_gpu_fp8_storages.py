"""Rows in 8 bits that a call returns: codes and scales are tensors of their own, which can be kept, saved and written apart from each other."""
from __future__ import annotations

import io

import pytest
import torch

import fp8_exact as X
from test_gpu_fp8 import weight

pytestmark = pytest.mark.gpu


def calls(ops):
    from orin_qwen_lossless_amd import torch_ops  # noqa: F401

    B = torch.ops.bf16n
    a = torch.randn((5, 272), device="cuda").to(torch.bfloat16)
    w = weight(ops, *X.matrix(48, 272, 1))
    rows = lambda r: (r.codes, r.scales)  # noqa: E731
    norm = ops.add_rmsnorm_fp8(a, want_sum=True, want_norm=True)
    stack = weight(ops, *X.matrix(48, 272, 2, 4), 4)
    ids = torch.randint(0, 4, (5, 2), device="cuda")
    return {"norm": (*rows(norm[0]), *norm[1:]), "norm alone": rows(ops.add_rmsnorm_fp8(a)), "rows": rows(ops.fp8_quantize_rows(a)), "gated": rows(ops.fp8_linear_glu2(a, w, w, X.E4M3)),
            "by expert": rows(ops.fp8_moe_mm_ids(a, ids, stack, 4, stack, X.E4M3)), "registered norm": B.add_rmsnorm_fp8(a, None, None, None, None, None, 1e-6),
            "registered rows": B.fp8_quantize_rows(a)}


def test_no_storage_is_shared(ops):
    for name, tensors in calls(ops).items():
        assert len({t.untyped_storage().data_ptr() for t in tensors}) == len(tensors), name
        for t in tensors:
            assert t.storage_offset() == 0 and t.untyped_storage().nbytes() == t.numel() * t.element_size() and not t.requires_grad, name
        assert tensors[1].stride() == (1, tensors[0].shape[0]) and tensors[1].dtype is torch.float32, name


def test_they_can_be_saved_and_written_apart(ops):
    for name, (codes, scales, *_) in calls(ops).items():
        f = io.BytesIO()
        torch.save((codes, scales), f)
        f.seek(0)
        c, s = torch.load(f, weights_only=True)
        assert torch.equal(c.view(torch.uint8), codes.view(torch.uint8)) and torch.equal(s, scales), name
        before = scales.clone()
        codes.view(torch.uint8).fill_(1)
        assert torch.equal(scales, before), name
        scales.mul_(2)
        assert (codes.view(torch.uint8) == 1).all() and torch.equal(scales, before * 2), name
