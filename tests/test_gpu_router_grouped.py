"""The selection with scores, a bias and groups against its definition in 64 bits: ids equal, weights within the rounding of FP32."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def exact(logits, k, bias, n_groups, topk_groups, scoring, group_score, renorm, scale):
    """One token at a time, by sorting (value, -index)."""
    rows_w, rows_i = [], []
    for z in logits.double():
        z = torch.where(z.isnan(), -math.inf, z)
        if scoring == "sigmoid":
            p = torch.sigmoid(z)
        else:
            m = z.max()
            p = torch.zeros_like(z) if m == -math.inf else torch.where(z == m, 1.0, torch.exp(z - m))
            p = p / p.sum() if p.sum() > 0 else p
        c = torch.where(z == -math.inf, -math.inf, p if bias is None else p + bias.double())
        c = torch.where(c.isnan(), -math.inf, c).tolist()
        E = len(c)
        size = E // n_groups
        rank = []
        for g in range(n_groups):
            best = sorted(c[g * size: (g + 1) * size], reverse=True)
            r = best[0] + best[1] if group_score == "top2" and size > 1 else best[0]
            rank.append(-math.inf if math.isnan(r) else r)
        kept = set(sorted(range(n_groups), key=lambda g: (-rank[g], g))[:topk_groups])
        ids = sorted((e for e in range(E) if e // size in kept), key=lambda e: (-c[e], e))[:k]
        w = [p[e].item() for e in ids]
        if renorm:
            t = sum(w)
            w = [v / t if t > 0 else 0.0 for v in w]
        rows_w.append([v * scale for v in w])
        rows_i.append(ids)
    return torch.tensor(rows_w, dtype=torch.float64).view(-1, k), torch.tensor(rows_i, dtype=torch.int32).view(-1, k)


def compare(ops, logits, k, bias=None, n_groups=1, topk_groups=None, scoring="softmax", group_score="max", renorm=True, scale=1.0):
    wts, ids = ops.router_topk_grouped(logits.cuda(), k, None if bias is None else bias.cuda(), n_groups, topk_groups, scoring, group_score, renorm, scale)
    w, i = exact(logits, k, bias, n_groups, n_groups if topk_groups is None else topk_groups, scoring, group_score, renorm, scale)
    assert torch.equal(ids.cpu(), i)
    # 64-bit arithmetic, rounded once to FP32 (the scale is FP32 already)
    assert ((wts.cpu().double() - w).abs() <= 2.0 ** -24 * (1 + 1e-6) * w.abs() + 2.0 ** -149).all()


@pytest.mark.parametrize("T,E,k,n_groups,topk_groups", [(1, 256, 8, 8, 4), (5, 64, 6, 1, 1), (3, 1, 1, 1, 1), (70, 96, 6, 6, 3), (9, 384, 12, 12, 5),
                                                       (4, 1024, 64, 64, 40), (130, 160, 7, 4, 4), (2, 513, 3, 27, 2), (6, 48, 2, 48, 2), (33, 128, 64, 2, 1)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_choice_and_weights(ops, T, E, k, n_groups, topk_groups, scoring):
    g = torch.Generator().manual_seed(T + E)
    logits = torch.randn((T, E), generator=g) * 2
    bias = torch.randn(E, generator=g) * 0.1
    compare(ops, logits, k, None, n_groups, topk_groups, scoring, "max", True)
    compare(ops, logits, k, bias, n_groups, topk_groups, scoring, "top2", False, 2.5)
    compare(ops, logits, k, bias, n_groups, topk_groups, scoring, "max", True, 0.5)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_ties_and_masks(ops, scoring):
    """Equal logits (ties to the lower index), -inf and NaN among them, rows that leave nothing, infinite ones, a saturated score."""
    g = torch.Generator().manual_seed(1)
    rows = [torch.zeros(64), torch.full((64,), -math.inf), torch.full((64,), math.nan), torch.randint(-2, 3, (64,), generator=g).float(),
            torch.where(torch.arange(64) < 61, -math.inf, 1.0), torch.full((64,), torch.finfo(torch.float32).min), torch.full((64,), 60.0)]
    r = torch.randn(64, generator=g)
    r[::3] = math.nan
    r[1::3] = -math.inf
    rows += [r, torch.where(torch.arange(64) % 7 == 3, math.inf, r), torch.where(torch.arange(64) < 32, -math.inf, 0.25)]
    logits = torch.stack(rows)
    bias = torch.zeros(64)
    bias[5], bias[6], bias[40] = math.inf, -math.inf, math.nan
    for gs in ("max", "top2"):
        for b in (None, bias):
            for n, kept in ((1, 1), (8, 2), (8, 8)):
                compare(ops, logits, 8, b, n, kept, scoring, gs)


def test_near_ties(ops):
    """Choices that differ by far less than a rounding of 32 bits, of sums with a bias."""
    E = 128
    base = torch.linspace(0.0, 1e-7, E)
    logits = base[torch.randperm(E, generator=torch.Generator().manual_seed(2))][None].repeat(3, 1).contiguous()
    compare(ops, logits, 16, torch.full((E,), 3.0), 4, 2, "sigmoid", "top2")
    compare(ops, logits, 16, torch.full((E,), 3.0), 4, 2, "softmax", "max")


def test_into_wider_rows(ops):
    g = torch.Generator().manual_seed(3)
    logits = torch.randn((7, 40), generator=g)
    wide = torch.randn((7, 100), generator=g)
    wide[:, 10:50] = logits
    wts, ids = torch.full((7, 9), 5.0, device="cuda"), torch.full((7, 9), 99, dtype=torch.int32, device="cuda")
    ops.router_topk_grouped(wide.cuda()[:, 10:50], 8, n_groups=4, topk_groups=2, out=(wts, ids))
    w, i = exact(logits, 8, None, 4, 2, "softmax", "max", True, 1.0)
    assert torch.equal(ids[:, :8].cpu(), i) and (ids[:, 8] == 99).all() and (wts[:, 8] == 5).all()
    assert ops.router_topk_grouped(torch.empty((0, 40), device="cuda"), 8)[1].shape == (0, 8)


def test_refusals(ops):
    lg = torch.zeros((2, 64), device="cuda")
    for kw in ({"k": 0}, {"k": 65}, {"k": 9, "n_groups": 8, "topk_groups": 1}, {"k": 2, "n_groups": 7}, {"k": 2, "n_groups": 8, "topk_groups": 9},
               {"k": 2, "n_groups": 8, "topk_groups": 0}, {"k": 2, "scoring": "relu"}, {"k": 2, "group_score": "mean"},
               {"k": 2, "bias": torch.zeros(63, device="cuda")}, {"k": 2, "bias": torch.zeros(64)}, {"k": 2, "bias": torch.zeros(64, device="cuda").half()}):
        with pytest.raises(ValueError):
            ops.router_topk_grouped(lg, **kw)
    for bad in (lg.half(), lg.cpu(), lg[0], lg.t()):
        with pytest.raises(ValueError):
            ops.router_topk_grouped(bad, 1)
    with pytest.raises(ValueError):
        ops.router_topk_grouped(torch.zeros((1, 1025), device="cuda"), 1)
