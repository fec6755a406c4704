"""Routed experts on 4-bit weights with FP32 activations: the type alone, not the number of tokens, decides what is taken and what the
hidden rows are held in."""
from __future__ import annotations

import pytest
import torch

import int4_exact as X
from test_gpu_int4 import acts, experts_exact, weight

pytestmark = pytest.mark.gpu


def layer(ops, E, mid, K, group):
    return [weight(ops, E * r, c, group, 300 + i) for i, (r, c) in enumerate(((mid, K), (mid, K), (K, mid)))]


@pytest.mark.parametrize("E,mid,K,T,n_used,group", [(8, 64, 256, 4, 2, 64), (8, 64, 256, 5, 2, 64), (8, 96, 128, 60, 3, 32), (3, 32, 160, 33000, 2, 128)])
@pytest.mark.parametrize("native", [True, False])
def test_any_number_of_pairs(ops, monkeypatch, E, mid, K, T, n_used, group, native):
    """At, just beyond and far beyond a pair to an expert, and beyond the columns of one launch; FP32 between the products in all of them."""
    if not native:
        monkeypatch.setattr(ops, "_host_calls", ops._NoNativeCalls)
    ms = layer(ops, E, mid, K, group)
    g = torch.Generator().manual_seed(T)
    ids = torch.randint(0, E, (T, n_used), generator=g, dtype=torch.int32)
    ids[-1, -1] = -1  # names no expert
    wts = torch.rand((T, n_used), generator=g) + 0.1
    x = acts(T, K, 303, torch.float32)
    y, b = experts_exact(x, [m for m, _ in ms], E, ids, wts, False)
    got = ops.int4_moe_experts_rows(x.cuda(), *(d for _, d in ms), ids.cuda(), E)
    assert got.shape == (T, n_used, K) and got.dtype is torch.float32 and not got[-1, -1].any()
    X.check((got.cpu().double() * wts.double()[:, :, None]).sum(1), y, b)
    if T <= 65535:
        X.check(ops.int4_moe_experts(x.cuda(), *(d for _, d in ms), wts.cuda(), ids.cuda(), E), y, X.rounded(y, b, torch.bfloat16))


def test_in_a_graph(ops):
    """Beyond a pair to an expert, captured and replayed with other activations and ids."""
    E, K, T = 4, 128, 40
    ds = [d for _, d in layer(ops, E, 64, K, 32)]
    x, ids = acts(T, K, 304, torch.float32).cuda(), torch.zeros((T, 2), dtype=torch.int32, device="cuda")
    wts = torch.ones((T, 2), device="cuda")
    ops.int4_moe_experts(x, *ds, wts, ids, E)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.int4_moe_experts(x, *ds, wts, ids, E)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.int4_moe_experts(x, *ds, wts, ids, E)
    for i in range(3):
        x.copy_(acts(T, K, 305 + i, torch.float32))
        ids.copy_(torch.randint(0, E, (T, 2), generator=torch.Generator().manual_seed(i), dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.int4_moe_experts(x, *ds, wts, ids, E))
