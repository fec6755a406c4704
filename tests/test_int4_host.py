"""4-bit weights with group scales, without a GPU: what their class and the calls refuse, quantization, and the shapes under tracing."""
from __future__ import annotations

import pytest
import torch

import int4_exact as X
from orin_qwen_lossless_amd import ops, torch_ops  # noqa: F401


def parts(rows=6, K=128, group=64):
    return X.make(rows, K, group, 1)


def test_the_weights_class_refuses_what_the_kernels_do_not_take():
    c, s, z = parts()
    w = ops.Int4Weight(c, s, z, 64)
    assert (w.rows, w.K, w.nbytes) == (6, 128, c.numel() + 2 * s.numel() + z.numel())
    assert ops.Int4Weight(c, s[:, :1].contiguous(), None, 128).zeros is None
    for bad in ((c.int(), s, z, 64), (c[:, ::2], s, z, 64), (c.reshape(-1), s, z, 64), (c[:, :24].contiguous(), s, z, 64), (c, s.float(), z, 64), (c, s[:5], z, 64),
                (c, s, z[:, :1].contiguous(), 64), (c, s, z.int(), 64), (c, s, z, 32), (c, s, z, 48), (c, s, z, 16), (c, s, z, 64.0),
                (torch.zeros((2, 8224), dtype=torch.uint8), torch.zeros((2, 129), dtype=torch.bfloat16), None, 128),
                (c, s.t().contiguous().t(), z, 64)):
        with pytest.raises(ValueError):
            ops.Int4Weight(*bad)


def test_calls_refuse_host_tensors():
    w = ops.Int4Weight(*parts(), 64)
    x, ids = torch.zeros((2, 128), dtype=torch.bfloat16), torch.zeros((2, 1), dtype=torch.int32)
    for call in (lambda: ops.int4_mmv(x, w), lambda: ops.int4_mmv_glu2(x, w, w), lambda: ops.int4_linear(x, w), lambda: ops.int4_route(ids, 2),
                 lambda: ops.int4_moe_mm_ids(x, ids, w, 2), lambda: ops.int4_moe_experts(x, w, w, w, torch.ones((2, 1)), ids, 2),
                 lambda: ops.router_topk_grouped(torch.zeros((2, 8)), 2)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("symmetric", [True, False])
def test_quantize_values(symmetric):
    """Weights that are codes already come back as they are; a group of zeros and one of a single value, too."""
    g = torch.Generator().manual_seed(2)
    u = torch.randint(-7, 8, (5, 96), generator=g).float()
    u[:, 0::32], u[:, 1::32] = 7, -7  # every group has its ends
    u[2, 32:64] = 0
    w = (u * 0.25).to(torch.bfloat16)
    q = ops.int4_quantize(w, 32, symmetric)
    code, s, z = X.parts(q.codes, q.scales, q.zeros, 32)
    got = s * (code - z)
    if symmetric:
        assert torch.equal(got, w.double())
    else:  # 14 steps of 0.25 on 15: half a step, the zero point's rounding and the scale's
        assert ((got - w.double()).abs() <= s * 1.0 + 15 * 2.0 ** -8 * s).all() and not got[2, 32:64].any()
    assert ops.int4_quantize(w.view(5, 3, 32), 32, symmetric).rows == 15


def test_quantize_refusals():
    for bad in (lambda: ops.int4_quantize(torch.zeros(64)), lambda: ops.int4_quantize(torch.zeros((2, 48))), lambda: ops.int4_quantize(torch.zeros((2, 64)).half()),
                lambda: ops.int4_quantize(torch.zeros((2, 64)), 24), lambda: ops.int4_quantize(torch.zeros((2, 64)), scale_dtype=torch.float32)):
        with pytest.raises(ValueError):
            bad()


def test_shapes_under_tracing():
    B = torch.ops.bf16n
    with torch._subclasses.FakeTensorMode():
        e = lambda *s, d=torch.bfloat16: torch.empty(s, dtype=d, device="cuda")  # noqa: E731
        m = lambda r, k: [e(r, k // 2, d=torch.uint8), e(r, k // 64)]  # noqa: E731
        y = B.int4_linear(e(2, 3, 128), *m(40, 128), None, 64, None)
        assert y.shape == (2, 3, 40) and y.dtype == torch.bfloat16
        y = B.int4_moe_experts(e(7, 128), m(4 * 64, 128), m(4 * 64, 128), m(4 * 128, 64), 64, e(7, 2, d=torch.float32), e(7, 2, d=torch.int32), 4)
        assert y.shape == (7, 128) and y.dtype == torch.bfloat16
        wts, ids = B.router_topk_grouped(e(7, 32, d=torch.float32), 4, None, 4, 2, "sigmoid", "top2", True, 1.0)
        assert wts.shape == ids.shape == (7, 4) and wts.dtype == torch.float32 and ids.dtype == torch.int32


@pytest.mark.parametrize("rows,K,group", [(64, 64, 1 << 20), (300, 2080, 1 << 11), (3, 96, 1 << 30)])
def test_quantize_takes_no_more_memory_for_wide_groups(rows, K, group, monkeypatch):
    """A group past the last column is that row's columns alone: the largest temporary is a piece, whatever the group."""
    from torch.utils._python_dispatch import TorchDispatchMode

    monkeypatch.setattr(ops, "DEQUANT_CHUNK_BYTES", 1 << 18)
    most = [0]

    class Sizes(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            out = func(*args, **(kwargs or {}))
            for t in out if isinstance(out, (tuple, list)) else (out,):
                if isinstance(t, torch.Tensor):
                    assert t.numel() <= limit, (func, t.shape)
                    most[0] = max(most[0], t.numel())
            return out

    w = torch.randn((rows, K), generator=torch.Generator().manual_seed(3))
    limit = max(rows * K, (1 << 18) // 4, -(-K // group) * min(group, 4096))
    for symmetric in (True, False):
        with Sizes():
            q = ops.int4_quantize(w, group, symmetric)
        assert q.group == group and q.scales.shape == (rows, -(-K // group))
        if group >= K:  # one group to a row: the same as with the smallest such group
            same = ops.int4_quantize(w, 1 << (K - 1).bit_length(), symmetric)
            assert torch.equal(q.codes, same.codes) and torch.equal(q.scales, same.scales)
            assert symmetric or torch.equal(q.zeros, same.zeros)
    assert most[0] > 0


def test_quantize_refuses_groups_that_no_weight_has():
    for group in (1 << 31, 64.0, 0, -32):
        with pytest.raises(ValueError):
            ops.int4_quantize(torch.zeros((2, 64)), group)


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("top,scale_dtype", [(1e6, torch.float16), (3e38, torch.bfloat16), (3e38, torch.float16)])
def test_quantize_of_weights_past_the_scales_range(symmetric, top, scale_dtype):
    """Finite weights give finite ones, the nearest codes of the largest scale there is; other groups do not notice.  A group with a
    weight that is not finite has no values."""
    w = torch.zeros((2, 96))
    w[0, 3], w[0, 5], w[1, 40] = top, -top, 2.0
    q = ops.int4_quantize(w, 32, symmetric, scale_dtype)
    code, s, z = X.parts(q.codes, q.scales, q.zeros, 32)
    got = s * (code - z)
    assert torch.isfinite(got).all() and got[0, 3] > 0 > got[0, 5] and abs(got[1, 40] - 2.0) <= 2.0 * 2.0 ** -8
    largest = torch.finfo(scale_dtype).max
    assert s[0, 0] == largest if top / 7.5 > largest else (got[0, 3] >= 0.9 * top and got[0, 5] <= -0.8 * top)
    w[0, 3] = float("inf")
    q = ops.int4_quantize(w, 32, symmetric, scale_dtype)
    code, s, z = X.parts(q.codes, q.scales, q.zeros, 32)
    assert not torch.isfinite(s[0, :32]).any() and torch.isfinite(s[0, 32:]).all()


def test_native_calls_of_an_older_build_are_not_used(monkeypatch):
    """An extension module of this torch's that was built before these calls came in: everything goes the general way, with a warning."""
    import types

    stale = types.SimpleNamespace(built_for=ops.torch_release(), bind=lambda *_: None, mmv=lambda *_: None, linear=lambda *_: None)
    monkeypatch.setattr(ops.importlib, "import_module", lambda *_: stale)
    monkeypatch.setattr(ops, "_host_calls", None)
    with pytest.warns(RuntimeWarning, match="native part"):
        assert ops._host() is ops._NoNativeCalls
    assert ops._host().int4_mmv(None, None, None, False, 32) is None
