"""Products with 4-bit weights and group scales against their definition in 64 bits (int4_exact: the bounds are derived there)."""
from __future__ import annotations

import pytest
import torch

import int4_exact as X

pytestmark = pytest.mark.gpu


def weight(ops, rows, K, group, seed, zeros=True, f16=False):
    m = X.make(rows, K, group, seed, zeros, f16)
    return (*m, group), ops.Int4Weight(*(None if t is None else t.cuda() for t in m), group)


def acts(tokens, K, seed, dtype=torch.bfloat16):
    return torch.randn((tokens, K), generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("rows,K,tokens,group", [
    (1, 32, 1, 32), (15, 64, 2, 64), (17, 96, 3, 32), (33, 160, 5, 128), (256, 2048, 1, 128), (512, 2048, 16, 128), (300, 2048, 17, 64),
    (129, 2080, 33, 32), (70, 4096, 7, 256), (64, 512, 64, 512), (31, 1024, 100, 128), (40, 9600, 4, 4096), (20, 16384, 6, 64), (5000, 256, 1, 64),
    (2500, 640, 20, 128), (9000, 160, 3, 32), (16500, 96, 20, 64), (8700, 320, 40, 128), (4200, 2048, 4, 256), (70, 4160, 200, 64)])
@pytest.mark.parametrize("zeros,f16", [(True, False), (False, True)])
def test_dense(ops, rows, K, tokens, group, zeros, f16):
    w, dw = weight(ops, rows, K, group, rows + K, zeros, f16)
    for dtype in (torch.bfloat16, torch.float32):
        x = acts(tokens, K, tokens, dtype)
        y, b = X.product(x, w)
        for out in (torch.float32, torch.bfloat16):
            X.check(ops.int4_mmv(x.cuda(), dw, out_dtype=out), y, X.rounded(y, b, out), (dtype, out))
        w2, dw2 = weight(ops, rows, K, group, rows + K + 1, zeros, not f16)  # (gate and up may differ in the scales' type)
        h, hb = X.gated(y, b, *X.product(x, w2))
        X.check(ops.int4_mmv_glu2(x.cuda(), dw, dw2), h, hb, dtype)


@pytest.mark.parametrize("rows,K,tokens,group", [(5, 64, 1, 32), (130, 2048, 9, 128), (257, 1056, 130, 64), (512, 2048, 517, 128), (1000, 512, 300, 32),
                                                 (4100, 1056, 200, 64), (2050, 160, 3000, 128), (8300, 416, 70, 32), (1030, 4128, 1100, 32), (640, 2080, 4100, 512)])
def test_linear(ops, rows, K, tokens, group):
    w, dw = weight(ops, rows, K, group, 3)
    x = acts(tokens, K, 4)
    y, b = X.product(x, w)
    X.check(ops.int4_linear(x.cuda(), dw), y, X.rounded(y, b, torch.bfloat16))
    bias = torch.randn(rows).to(torch.bfloat16)
    yb = y + bias.double()
    X.check(ops.int4_linear(x.cuda(), dw, bias.cuda()), yb, X.rounded(yb, b + X.STEP32 * yb.abs(), torch.bfloat16), "bias")


def test_linear_takes_views(ops):
    """Rows apart by more than their length, leading axes, rows that are not 16-byte aligned, no tokens."""
    w, dw = weight(ops, 48, 128, 64, 5)
    wide = acts(6, 300, 6).cuda()
    for x in (wide[:, :128], wide[:, 8:136], wide[:, 3:131], wide.view(2, 3, 300)[..., :128], wide[:0, :128]):
        y, b = X.product(x.reshape(-1, 128), w)
        got = ops.int4_linear(x, dw)
        assert got.shape == (*x.shape[:-1], 48)
        if x.numel():
            X.check(got.reshape(-1, 48), y, X.rounded(y, b, torch.bfloat16))


@pytest.mark.parametrize("E,N,K,T,n_used,group", [(4, 32, 64, 1, 2, 32), (16, 48, 512, 3, 4, 128), (8, 100, 2048, 2, 8, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_expert_columns(ops, E, N, K, T, n_used, group, dtype):
    w, dw = weight(ops, E * N, K, group, 7)
    w2, dw2 = weight(ops, E * N, K, group, 8)
    g = torch.Generator().manual_seed(9)
    ids = torch.randint(0, E, (T, n_used), generator=g, dtype=torch.int32)
    ids[0, 0], ids[-1, -1] = -1, E  # no such expert
    for x in (acts(T, K, 10, dtype), acts(T * n_used, K, 11, dtype).view(T, n_used, K)):
        xp = x[:, None].expand(T, n_used, K) if x.dim() == 2 else x
        for idt in (torch.int32, torch.int64):
            got = ops.int4_mmv(x.cuda(), dw, ids.to(idt).cuda(), N)
            glu = ops.int4_mmv_glu2(x.cuda(), dw, dw2, ids.to(idt).cuda(), N, torch.bfloat16)
            for t in range(T):
                for i in range(n_used):
                    e = int(ids[t, i])
                    if not 0 <= e < E:
                        assert not got[t, i].any() and not glu[t, i].any()
                        continue
                    cut = lambda m: (*(None if p is None else p[e * N: e * N + N] for p in m[:3]), group)  # noqa: E731
                    y, b = X.product(xp[t, i: i + 1], cut(w))
                    X.check(got[t, i: i + 1], y, b)
                    h, hb = X.gated(y, b, *X.product(xp[t, i: i + 1], cut(w2)))
                    X.check(glu[t, i: i + 1], h, X.rounded(h, hb, torch.bfloat16))


@pytest.mark.parametrize("E,T,n_used", [(1, 1, 1), (5, 3, 2), (256, 77, 8), (300, 1, 8), (16, 700, 6), (3, 5000, 4)])
def test_route(ops, E, T, n_used):
    ids = torch.randint(-1, E + 1, (T, n_used + 2), generator=torch.Generator().manual_seed(T))
    for idt in (torch.int32, torch.int64):
        use = ids.to(idt).cuda()[:, 1: 1 + n_used]
        if idt is torch.int64:
            use = use.clone()
            use[0, 0] += 1 << 32  # an expert only in its lower half
        pairs, bounds = ops.int4_route(use, E)
        flat = use.cpu().reshape(-1).long()
        flat = torch.where((flat >= 0) & (flat < E), flat, E)
        want = torch.sort(flat, stable=True)
        assert torch.equal(pairs.cpu().long(), want.indices)
        assert torch.equal(bounds.cpu().long(), torch.searchsorted(want.values, torch.arange(E + 2)))


@pytest.mark.parametrize("E,N,K,T,n_used,group", [(8, 48, 128, 1, 1, 32), (8, 48, 256, 40, 2, 64), (16, 64, 512, 300, 4, 128), (5, 33, 96, 7, 3, 32), (2, 160, 2048, 700, 2, 128)])
def test_batched_experts(ops, E, N, K, T, n_used, group):
    w, dw = weight(ops, E * N, K, group, 12)
    w2, dw2 = weight(ops, E * N, K, group, 13, f16=True)
    g = torch.Generator().manual_seed(14)
    ids = torch.randint(0, E, (T, n_used), generator=g, dtype=torch.int32)  # a token may name an expert twice
    ids[T // 2, 0] = -1
    ids[-1, -1] = E + 3
    cut = lambda m, e: (*(None if p is None else p[e * N: e * N + N] for p in m[:3]), group)  # noqa: E731
    for x in (acts(T, K, 15), acts(T * n_used, K, 16).view(T, n_used, K)):
        xp = (x[:, None].expand(T, n_used, K) if x.dim() == 2 else x).reshape(-1, K)
        for out in (torch.float32, torch.bfloat16):
            got = ops.int4_moe_mm_ids(x.cuda(), ids.cuda(), dw, E, out_dtype=out).reshape(-1, N)
            glu = ops.int4_moe_mm_ids(x.cuda(), ids.cuda(), dw, E, up=dw2, out_dtype=out).reshape(-1, N)
            for e in range(E):
                at = (ids.reshape(-1) == e).nonzero()[:, 0]
                if len(at):
                    y, b = X.product(xp[at], cut(w, e))
                    X.check(got[at.cuda()], y, X.rounded(y, b, out))
                    h, hb = X.gated(y, b, *X.product(xp[at], cut(w2, e)))
                    X.check(glu[at.cuda()], h, X.rounded(h, hb, out))
            none = ((ids < 0) | (ids >= E)).reshape(-1).cuda()
            assert not got[none].any() and not glu[none].any()


def experts_exact(x, ws, E, ids, wts, batched):
    """(moe_experts' result, bound) with the roundings of either path"""
    K, T = x.shape[1], x.shape[0]
    (gate, up, down), n = ws, ids.shape[1]
    mid = gate[0].shape[0] // E
    y, b = torch.zeros((T, K), dtype=torch.float64), torch.zeros((T, K), dtype=torch.float64)
    for e in range(E):
        tok, slot = (ids == e).nonzero(as_tuple=True)
        if not len(tok):
            continue
        cut = lambda m, r: (*(None if p is None else p[e * r: e * r + r] for p in m[:3]), m[3])  # noqa: E731
        h, hb = X.gated(*X.product(x[tok], cut(gate, mid)), *X.product(x[tok], cut(up, mid)))
        if batched:
            hb = X.rounded(h, hb, torch.bfloat16)
        d = cut(down, K)
        o, ob = X.product(h, d)
        u, s, z = X.parts(*d)
        ob = ob * 1.01 + hb @ (s * (u - z)).abs().t()
        wt = wts[tok, slot].double()[:, None]
        y.index_add_(0, tok, o * wt)
        b.index_add_(0, tok, (ob + (n + 1) * X.STEP32 * o.abs()) * wt)
    return y, b


@pytest.mark.parametrize("T", [1, 4, 50])
def test_router_and_experts_together(ops, T):
    """The selection in groups, then the experts that it named, as a layer runs them, eagerly and as a captured graph."""
    E, mid, K, k, group = 32, 64, 256, 4, 64
    ms = [weight(ops, E * r, c, group, 20 + i) for i, (r, c) in enumerate(((mid, K), (mid, K), (K, mid)))]
    x = acts(T, K, 24)
    logits = torch.randn((T, E), generator=torch.Generator().manual_seed(25))
    bias = torch.randn(E, generator=torch.Generator().manual_seed(26)) * 0.1
    xd, ld, bd = x.cuda(), logits.cuda(), bias.cuda()

    def layer():
        wts, ids = ops.router_topk_grouped(ld, k, bias=bd, n_groups=4, topk_groups=2, scoring="sigmoid", group_score="top2")
        return wts, ids, ops.int4_moe_experts(xd, *(d for _, d in ms), wts, ids, E)

    wts, ids, got = layer()
    y, b = experts_exact(x, [m for m, _ in ms], E, ids.cpu(), wts.cpu(), ops.int4_moe_experts_batched(T, k, E))
    X.check(got, y, X.rounded(y, b, torch.bfloat16))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = layer()
    for i in range(3):
        ld.copy_(torch.randn((T, E), generator=torch.Generator().manual_seed(30 + i)))
        xd.copy_(acts(T, K, 40 + i))
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip(again, layer()):
            assert torch.equal(a, e)


def test_same_bits_again(ops):
    _, dw = weight(ops, 4000, 2048, 128, 50)
    x = acts(20, 2048, 51).cuda()
    first = ops.int4_mmv(x, dw)
    assert all(torch.equal(first, ops.int4_mmv(x, dw)) for _ in range(5))


@pytest.mark.parametrize("rows,T", [(64, 5), (8400, 5), (4000, 300)])
def test_not_finite(ops, rows, T):
    """An activation that is not finite reaches every result of its own column and no other; so does a scale its row."""
    _, dw = weight(ops, rows, 256, 64, 52)
    others = torch.arange(T) != 2
    for dtype in (torch.bfloat16, torch.float32):
        for bad in (float("inf"), float("-inf"), float("nan")):
            x = acts(T, 256, 53, dtype)
            x[2, 77] = bad
            y = ops.int4_mmv(x.cuda(), dw)
            assert not torch.isfinite(y[2]).any() and torch.isfinite(y[others]).all()
    dw.scales[7, 1] = float("nan")
    y = ops.int4_mmv(acts(T, 256, 54).cuda(), dw)
    assert torch.isnan(y[:, 7]).all() and torch.isfinite(y[:, torch.arange(rows) != 7]).all()


def test_nothing_to_do(ops):
    """No tokens, no slots, no rows."""
    w, up, down = (weight(ops, 4 * r, c, 32, 63 + i)[1] for i, (r, c) in enumerate(((32, 64), (32, 64), (64, 32))))
    x, ids, wts = acts(3, 64, 66).cuda(), torch.zeros((3, 2), dtype=torch.int32, device="cuda"), torch.ones((3, 2), device="cuda")
    assert ops.int4_moe_experts(x[:0], w, up, down, wts[:0], ids[:0], 4).shape == (0, 64)
    assert not ops.int4_moe_experts(x, w, up, down, wts[:, :0].contiguous(), ids[:, :0], 4).any()
    assert ops.int4_mmv(x[:0], w).shape == (0, 128) and ops.int4_moe_mm_ids(x[:0], ids[:0], w, 4).shape == (0, 2, 32)
    assert ops.int4_mmv(x, ops.Int4Weight(w.codes[:0], w.scales[:0], w.zeros[:0], 32)).shape == (3, 0)
    pairs, bounds = ops.int4_route(ids[:0], 4)
    assert pairs.numel() == 0 and not bounds.any() and bounds.numel() == 6


def test_large_and_small_f32(ops):
    """FP32 activations keep all their bits over the range of exponents."""
    w, dw = weight(ops, 32, 256, 64, 55)
    for scale in (1e-30, 1.0, 1e30):
        x = acts(3, 256, 56, torch.float32) * scale
        y, b = X.product(x, w)
        X.check(ops.int4_mmv(x.cuda(), dw), y, b, scale)


def test_other_stream(ops):
    w, dw = weight(ops, 300, 512, 64, 57)
    x = acts(9, 512, 58)
    y, b = X.product(x, w)
    s = torch.cuda.Stream()
    xd = x.cuda()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.int4_mmv(xd, dw)
    s.synchronize()
    X.check(got, y, b)


def test_with_and_without_the_native_calls(ops, monkeypatch):
    """The calls from Python in native code and the general way launch the same kernels; both refuse the same."""
    E, mid, K, group = 8, 64, 128, 32
    w, up, down = (weight(ops, E * r, c, group, 70 + i)[1] for i, (r, c) in enumerate(((mid, K), (mid, K), (K, mid))))
    x, logits = acts(30, K, 73).cuda(), torch.randn((30, E), generator=torch.Generator().manual_seed(74)).cuda()
    wts, ids = ops.router_topk_grouped(logits, 2)

    def results():
        out = []
        for a in (x, x[:3], x[:, :].float()[:5]):
            out += [ops.int4_mmv(a, w), ops.int4_mmv(a, w, out_dtype=torch.bfloat16), ops.int4_mmv_glu2(a, w, up)]
        out += [ops.int4_linear(x, w), ops.int4_linear(torch.cat([x] * 40), weight(ops, 4000, K, group, 75)[1])]
        for t in (1, 3, 30):
            for i, v in ((ids, wts), (ids.long(), wts.bfloat16())):
                out.append(ops.int4_moe_experts(x[:t], w, up, down, v[:t].contiguous(), i[:t], E))
        for kw in ({}, {"bias": logits[0].contiguous(), "n_groups": 4, "topk_groups": 2, "scoring": "sigmoid", "group_score": "top2", "renorm": False, "scale": 2.0}):
            out += ops.router_topk_grouped(logits, 3, **kw)
        return out

    native = results()
    with pytest.raises(ValueError):
        ops.router_topk_grouped(logits, 3, n_groups=3)
    monkeypatch.setattr(ops, "_host_calls", ops._NoNativeCalls)
    for a, b in zip(native, results(), strict=True):
        assert a.dtype == b.dtype and torch.equal(a, b)
    with pytest.raises(ValueError):
        ops.router_topk_grouped(logits, 3, n_groups=3)


def test_registered_operators(ops):
    from orin_qwen_lossless_amd import torch_ops  # noqa: F401

    B = torch.ops.bf16n
    w, up, down = (weight(ops, 4 * r, c, 64, 80 + i)[1] for i, (r, c) in enumerate(((64, 128), (64, 128), (128, 64))))
    x, logits = acts(5, 128, 83).cuda(), torch.randn((5, 4), generator=torch.Generator().manual_seed(84)).cuda()
    wts, ids = B.router_topk_grouped(logits, 2, None, 1, 1, "softmax", "max", True, 1.0)
    assert all(torch.equal(a, b) for a, b in zip((wts, ids), ops.router_topk_grouped(logits, 2)))
    m = lambda t: [t.codes, t.scales, t.zeros]  # noqa: E731
    assert torch.equal(B.int4_linear(x, *m(w), 64, None), ops.int4_linear(x, w))
    assert torch.equal(B.int4_moe_experts(x, m(w), m(up), m(down), 64, wts, ids, 4), ops.int4_moe_experts(x, w, up, down, wts, ids, 4))


def test_results_between_strides_and_behind_stay(ops):
    """The C call with results further apart than their rows: what lies between and behind them is left as it was, in every kernel."""
    import ctypes as C

    from orin_qwen_lossless_amd import _lib

    for rows, K, T, ws in ((40, 128, 3, False), (9000, 64, 20, False), (5000, 128, 300, True)):
        w, dw = weight(ops, rows, K, 32, 90)
        x = acts(T, K, 91)
        xd, y = x.cuda(), torch.full((T + 1, rows + 24), 7.0, device="cuda")
        a = _lib.MmvArgs(x=xd.data_ptr(), y=y.data_ptr(), x_tok=K * 2, y_tok=y.stride(0) * 4, rows_per_matrix=rows, nrows=rows, ncols=T, n_used=1, x_per_slot=1,
                         x_bf16=1, y_bf16=0)
        cw = ops._c_int4(dw)
        space = ops._int4_workspace(cw, T, xd.device) if ws else None
        _lib.check(_lib.lib().bf16n_int4_mmv(C.byref(cw), None, C.byref(a), 0, space.data_ptr() if ws else None, space.numel() if ws else 0, ops._stream()))
        exact, bound = X.product(x, w)
        X.check(y[:T, :rows], exact, bound)
        assert (y[:T, rows:] == 7).all() and (y[T] == 7).all()


def test_codes_beyond_four_gigabytes(ops):
    """Places past 32 bits in the codes, for every kernel: the last rows of a large matrix are those of a small one."""
    rows, K, group = 560000, 16384, 4096
    g = torch.Generator(device="cuda").manual_seed(92)
    codes = torch.randint(0, 256, (rows, K // 2), generator=g, dtype=torch.uint8, device="cuda")
    scales = (torch.rand((rows, 4), generator=g, device="cuda") * 0.01).to(torch.bfloat16)
    big = ops.Int4Weight(codes, scales, None, group)
    tail = (codes[-64:].cpu(), scales[-64:].cpu(), None, group)
    for T in (1, 20):
        x = acts(T, K, 93)
        y, b = X.product(x, tail)
        X.check(ops.int4_mmv(x.cuda(), big)[:, -64:], y, b, T)
    E = rows // 64
    ids = torch.tensor([[E - 1, 0]] * 2, dtype=torch.int32, device="cuda")
    x = acts(2, K, 94)
    y, b = X.product(x, tail)
    X.check(ops.int4_mmv(x.cuda(), big, ids, 64)[:, 0], y, b, "ids")
    half = ops.Int4Weight(codes, scales, None, group)
    ids = torch.full((40, 1), 1, dtype=torch.int32, device="cuda")  # two matrices of 280000 rows, the second one named: many columns
    x = acts(40, K, 95)
    y, b = X.product(x, tail)
    X.check(ops.int4_moe_mm_ids(x.cuda(), ids, half, 2)[:, 0, -64:], y, b, "lists")


def test_activations_beyond_four_gigabytes(ops):
    """Activation rows so far apart that their places pass 32 bits: more columns than a pass has, all of them right."""
    w, dw = weight(ops, 6000, 128, 64, 96)
    far = torch.empty(70 * 35_000_000, dtype=torch.bfloat16, device="cuda").as_strided((70, 128), (35_000_000, 1))
    x = acts(70, 128, 97)
    far.copy_(x)
    y, b = X.product(x, w)
    X.check(ops.int4_mmv(far, dw), y, b)


@pytest.mark.parametrize("T", [1, 5])
def test_decode_step_with_experts_in_four_bits(ops, T):
    """A layer of the decode step with such experts: the router's choice, and the experts' rows, from its own input."""
    from orin_qwen_lossless_amd import decode_step as D
    from orin_qwen_lossless_amd import synth

    seed = [9000]

    def gen(rows, k):
        seed[0] += 1
        return synth.weights_torch(rows, k, seed[0], "cuda")

    sets, _, nbytes = D.make_layer_sets(ops, gen, 1, False, "int4")
    assert isinstance(sets[0]["gate"], ops.Int4Weight) and nbytes["gate"] == sets[0]["gate"].nbytes
    step = D.Bf16nStep(ops, sets, ops.int4_quantize(gen(512, D.K_MODEL)), 2, T)
    x2 = acts(T, D.K_MODEL, 98).cuda()
    ys, wts, ids = step.experts(sets[0], x2)
    w, i = ops.router_topk(ops.mmv(x2, sets[0]["router"]), D.TOPK)
    assert torch.equal(ids[:, :D.TOPK], i) and torch.equal(wts[:, :D.TOPK], w) and (ids[:, D.TOPK] == D.E).all()
    batched = ops.int4_moe_experts_batched(T, D.TOPK + 1, D.EA)
    cut = lambda m, e, n: (m.codes[e * n: e * n + n], m.scales[e * n: e * n + n], None, m.group)  # noqa: E731
    for t in range(T):
        for j in (0, D.TOPK):
            e = int(ids[t, j])
            h, hb = X.gated(*X.product(x2[t: t + 1], cut(sets[0]["gate"], e, D.N_MID)), *X.product(x2[t: t + 1], cut(sets[0]["up"], e, D.N_MID)))
            if batched:
                hb = X.rounded(h, hb, torch.bfloat16)
            d = cut(sets[0]["down"], e, D.K_MODEL)
            y, b = X.product(h, d)
            u, s, z = X.parts(*d)
            X.check(ys[t: t + 1, j], y, b * 1.01 + hb @ (s * (u - z)).abs().t(), (t, j))
    h = acts(T, D.K_MODEL, 99).cuda()
    graph, out = D.capture(step, h)
    for k in range(3):
        h.copy_(acts(T, D.K_MODEL, 100 + k))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step(h)) and out.shape == (T, 512)


def test_quantize(ops):
    """Codes are within half a step of the weight (and a rounding of the scale: the largest weight may lie past the last code by that)."""
    w = torch.randn((300, 1056), generator=torch.Generator().manual_seed(60)).mul_(0.02).to(torch.bfloat16)
    w[5, :64] = 0
    for symmetric in (True, False):
        for group in (32, 128, 2048):
            for dt, eps in ((torch.bfloat16, 2.0 ** -8), (torch.float16, 2.0 ** -11)):
                q = ops.int4_quantize(w.cuda(), group, symmetric, dt)
                u, s, z = X.parts(q.codes, q.scales, q.zeros, group)
                # fp16 scales below 2^-14 are denormal: a step of 2^-24
                slack = 15 * (eps * s.abs() + (2.0 ** -24 if dt is torch.float16 else 0))
                assert ((s * (u - z) - w.double()).abs() <= (0.5 if symmetric else 1.0) * s * (1 + 2.0 ** -20) + slack).all()
                assert not (s * (u - z))[5, :32].any()


def test_refusals(ops):
    _, dw = weight(ops, 64, 256, 64, 61)
    x = acts(4, 256, 62).cuda()
    ids = torch.zeros((4, 2), dtype=torch.int32, device="cuda")
    for call in (lambda: ops.int4_mmv(x.half(), dw), lambda: ops.int4_mmv(x[:, :128], dw), lambda: ops.int4_mmv(x.cpu(), dw),
                 lambda: ops.int4_mmv(x, dw, out_dtype=torch.float16), lambda: ops.int4_mmv(x, dw, rows_per_matrix=32),
                 lambda: ops.int4_mmv(x, dw, ids, 48), lambda: ops.int4_mmv(x, dw, ids[:3], 32), lambda: ops.int4_mmv(x, dw, ids.float(), 32),
                 lambda: ops.int4_mmv(x, dw, ids.cpu(), 32), lambda: ops.int4_mmv(x[None], dw),
                 lambda: ops.int4_mmv(torch.zeros(1028, device="cuda", dtype=torch.bfloat16)[4:].view(4, 256), dw),
                 lambda: ops.int4_mmv_glu2(x, dw, weight(ops, 32, 256, 64, 1)[1]), lambda: ops.int4_mmv_glu2(x, dw, weight(ops, 64, 256, 32, 1)[1]),
                 lambda: ops.int4_mmv_glu2(x, dw, weight(ops, 64, 256, 64, 1, False)[1]),
                 lambda: ops.int4_linear(x.float(), dw), lambda: ops.int4_linear(x[:, :32], dw),
                 lambda: ops.int4_moe_mm_ids(x, ids, dw, 3), lambda: ops.int4_moe_mm_ids(x.float(), ids, dw, 2),
                 lambda: ops.int4_moe_mm_ids(x, ids, dw, 2, routes=ops.int4_route(ids, 3)), lambda: ops.int4_route(ids[0], 2)):
        with pytest.raises(ValueError):
            call()
