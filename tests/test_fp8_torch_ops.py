"""The registered operators in 8-bit floating point under tracing, without a GPU: shapes, types and strides are those of the calls."""
from __future__ import annotations

import pytest
import torch

from orin_qwen_lossless_amd import decode_step, ops, torch_ops  # noqa: F401

E4M3 = torch.float8_e4m3fn


def test_shapes_under_tracing():
    B = torch.ops.bf16n
    with torch._subclasses.FakeTensorMode():
        e = lambda *s, d=torch.bfloat16: torch.empty(s, dtype=d, device="cuda")  # noqa: E731
        m = lambda r, k, n=1: [e(n * r, k, d=E4M3), e(n * -(-r // 128), -(-k // 128), d=torch.float32)]  # noqa: E731
        q, s = B.fp8_quantize_rows(e(5, 272))
        assert q.shape == (5, 272) and q.dtype is E4M3 and s.shape == (5, 3) and s.dtype is torch.float32 and s.stride() == (1, 5)
        q, s, total = B.add_rmsnorm_fp8(e(5, 272), None, None, None, None, None, 1e-6)
        assert q.shape == total.shape == (5, 272) and total.dtype is torch.bfloat16 and s.shape == (5, 3)
        y = B.fp8_linear(e(2, 3, 272), None, *m(40, 272), None, True)
        assert y.shape == (2, 3, 40) and y.dtype is torch.bfloat16
        assert B.fp8_linear(q, s, *m(40, 272), None, False).dtype is torch.float32
        y = B.fp8_linear_glu2(q, s, *m(48, 272), *m(48, 272), True)
        assert y.shape == (5, 48) and y.dtype is torch.bfloat16
        y = B.fp8_moe_experts(e(7, 128), None, m(64, 128, 4), m(64, 128, 4), m(128, 64, 4), e(7, 2, d=torch.float32), e(7, 2, d=torch.int32), 4)
        assert y.shape == (7, 128) and y.dtype is torch.bfloat16


def test_weights_of_a_step_in_8_bits():
    w = torch.randn((3 * 40, 272), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    got, nbytes = decode_step.encode_policy(ops, w, 3, "fp8")
    assert isinstance(got, ops.Fp8Weight) and got.n_matrices == 3 and nbytes == got.nbytes == 3 * (40 * 272 + 3 * 4)


def test_a_list_that_is_no_weight():
    with pytest.raises(ValueError):
        torch_ops._fp8([torch.zeros((4, 16))], 2)
