"""Operators in 8-bit floating point as they are used: one behind the other, in graphs, on other streams, from every way in, in the decode step, and every
kernel and tile that their sizes choose."""
from __future__ import annotations

import pytest
import torch

import fp8_exact as X
from test_gpu_fp8 import BF16_HALF, check, give, weight
from test_gpu_fp8_experts import by_pair, ids_for

pytestmark = pytest.mark.gpu


def names(kernel):
    name, _, numbers = kernel.partition("<")
    return name, [int(n) for n in numbers.rstrip(">").split(",")] if numbers else []


# (rows, K, tokens, results) -> what k_fp8_few or k_fp8_many are instances of
FEW = [(512, 2048, 1, 1, 8, 1), (512, 2048, 17, 2, 8, 1), (8000, 640, 3, 1, 8, 0), (4000, 1040, 32, 2, 8, 1), (512, 8192, 2, 1, 8, 0), (400, 8192, 31, 2, 8, 0), (512, 2048, 200, 2, 8, 1),
       (300, 9104, 70, 1, 8, 0), (16, 1040, 8000, 2, 8, 1)]


@pytest.mark.parametrize("R,K,T,ct,nw,one", FEW)
@pytest.mark.parametrize("kind", ["bf16", "f32", "rows"])
def test_every_form_for_few_columns(ops, R, K, T, ct, nw, one, kind):
    c, s = X.matrix(R, K, 11)
    x, q, xs = give(X.rows(T, K, 12), kind)
    got = ops.fp8_linear(x, weight(ops, c, s), out_dtype=torch.float32)
    name, numbers = names(ops.last_kernel())
    assert name == "k_fp8_few" and (numbers[0], numbers[3], numbers[4]) == (ct, nw, one), ops.last_kernel()
    check(got, *X.product(q, xs, c, s))
    check(ops.fp8_linear_glu2(x, weight(ops, c, s), weight(ops, c, s), torch.float32), *X.gated(*[*X.product(q, xs, c, s)] * 2))
    assert names(ops.last_kernel())[0] == "k_fp8_few"


# few columns of many rows: narrow tiles
NARROW = [(9000, 640, 3, 1), (9000, 144, 16, 1), (20000, 272, 2, 2), (90000, 144, 1, 2), (40000, 2576, 13, 2)]


@pytest.mark.parametrize("R,K,T,rt", NARROW)
@pytest.mark.parametrize("kind,out", [("bf16", torch.bfloat16), ("f32", torch.float32), ("rows", torch.float32), ("rows", torch.bfloat16)])
def test_narrow_tiles(ops, R, K, T, rt, kind, out):
    c, s = (t.cuda() for t in X.matrix(R, K, 48, bf16=kind == "f32"))
    x, q, xs = give(X.rows(T, K, 49), kind)
    got = ops.fp8_linear(x, ops.Fp8Weight(c, s), out_dtype=out)
    name, numbers = names(ops.last_kernel())
    assert name == "k_fp8_many" and numbers[:4] == [4, 1, rt, 1], ops.last_kernel()
    y, dy = X.product(q.cuda(), xs.cuda(), c, s, out)
    check(got, y.cpu(), dy.cpu())


@pytest.mark.parametrize("T,n_used,E,N,K,nw", [(8, 8, 128, 528, 272, 4), (1, 60, 64, 512, 64, 4), (60, 1, 64, 8000, 144, 4), (1, 2, 4, 512, 2048, 8)])
def test_single_pairs(ops, T, n_used, E, N, K, nw):
    (c, s), (cu, su) = X.matrix(N, K, 50, E), X.matrix(N, K, 51, E)
    ids = ids_for(T, n_used, E, 52)
    x, q, xs = give(X.rows(T, K, 53, False), "bf16")
    y, dy = by_pair(q, xs, c, s, ids, E, torch.float32)
    got = ops.fp8_moe_mm_ids(x, ids.cuda(), weight(ops, c, s, E), E)
    name, numbers = names(ops.last_kernel())
    assert name == "k_fp8_few" and numbers[3] == nw, ops.last_kernel()
    check(got.view(T * n_used, N), y, dy)
    y, dy = X.gated(y, dy, *by_pair(q, xs, cu, su, ids, E, torch.float32))
    check(ops.fp8_moe_mm_ids(x, ids.cuda(), weight(ops, c, s, E), E, weight(ops, cu, su, E)).view(T * n_used, N), y, dy)


MANY = [((8192, 272, 8192), torch.bfloat16, (2, 4, 8, 4)), ((2000, 144, 4096), torch.bfloat16, (2, 2, 4, 4)), ((5120, 272, 500), torch.bfloat16, (2, 2, 2, 2)), ((5120, 272, 1024), torch.bfloat16, (2, 2, 4, 2)),
        ((520, 272, 100), torch.bfloat16, (2, 2, 1, 2)), ((4096, 144, 4096), torch.float32, (4, 2, 4, 4)), ((5120, 272, 2050), torch.float32, (2, 2, 4, 2)), ((5120, 272, 150), torch.float32, (2, 2, 2, 2)),
        ((4096, 9104, 70), torch.float32, (2, 2, 1, 2)), ((4096, 9104, 70), torch.bfloat16, (2, 2, 1, 2))]


@pytest.mark.parametrize("shape,out,tile", MANY)
def test_every_tile_of_the_dense_product(ops, shape, out, tile):
    R, K, T = shape
    c, s = (t.cuda() for t in X.matrix(R, K, 13))
    q, xs = (t.cuda() for t in X.quantize(X.rows(T, K, 14)))
    got = ops.fp8_linear(ops.Fp8Rows(q, xs), ops.Fp8Weight(c, s), out_dtype=out)
    name, numbers = names(ops.last_kernel())
    assert name == "k_fp8_many" and tuple(numbers[:4]) == tile, ops.last_kernel()
    y, dy = X.product(q, xs, c, s, out)
    check(got, y.cpu(), dy.cpu())


# (rows, K, tokens) -> the tile of results that are codes, and of others
GATED = [((1024, 144, 2050), (4, 2, 4, 4), (2, 2, 4, 2)), ((2048, 144, 2050), (4, 1, 4, 2), (2, 2, 4, 2)), ((2048, 272, 700), (4, 2, 4, 2), (2, 2, 2, 2)), ((1408, 272, 500), (4, 1, 4, 1), (2, 2, 2, 2)),
         ((1408, 272, 100), (4, 1, 4, 1), (2, 2, 2, 2)), ((2064, 9104, 70), (4, 1, 4, 1), (2, 2, 2, 2)), ((2048, 144, 4096), (4, 2, 4, 4), (4, 2, 4, 4)), ((9008, 144, 9), (4, 1, 4, 1), (4, 1, 2, 1)),
         ((70000, 144, 3), (4, 1, 4, 1), (4, 1, 4, 1))]


@pytest.mark.parametrize("shape,codes,others", GATED)
@pytest.mark.parametrize("out", [X.E4M3, torch.bfloat16, torch.float32])
def test_every_tile_of_the_gated_product(ops, shape, codes, others, out):
    R, K, T = shape
    tile = codes if out is X.E4M3 else others
    (c, s), (cu, su) = ([t.cuda() for t in X.matrix(R, K, 15 + i)] for i in range(2))
    q, xs = (t.cuda() for t in X.quantize(X.rows(T, K, 17, False)))
    got = ops.fp8_linear_glu2(ops.Fp8Rows(q, xs), ops.Fp8Weight(c, s), ops.Fp8Weight(cu, su), out)
    name, numbers = names(ops.last_kernel())
    assert name == "k_fp8_many" and tuple(numbers[:4]) == tile, ops.last_kernel()
    y, dy = X.gated(*X.product(q, xs, c, s, out), *X.product(q, xs, cu, su, out))
    if out is X.E4M3:
        assert X.near_codes(got.codes, got.scales, y, dy)
    else:
        check(got, y.cpu(), dy.cpu())


@pytest.mark.parametrize("T,n_used,E,same", [(120, 2, 64, False), (400, 2, 64, True), (4000, 2, 16, False), (1700, 1, 3, True), (13, 1, 1, False), (97, 2, 2, False)])
def test_lists_of_every_length(ops, T, n_used, E, same):
    """Lists from none to more columns than a block's two turns have; `same`: every pair names one matrix."""
    mid, K = 144, 272
    (cg, sg), (cu, su), (cd, sd) = X.matrix(mid, K, 18, E), X.matrix(mid, K, 19, E), X.matrix(K, mid, 20, E)
    g, u, d = weight(ops, cg, sg, E), weight(ops, cu, su, E), weight(ops, cd, sd, E)
    ids = torch.full((T, n_used), E - 1) if same else ids_for(T, n_used, E, 21)
    dev = ids.cuda()
    x, q, xs = give(X.rows(T, K, 22, False), "rows")
    hidden = ops.fp8_moe_mm_ids(x, dev, g, E, u, X.E4M3)
    h, dh = X.gated(*by_pair(q, xs, cg, sg, ids, E, X.E4M3), *by_pair(q, xs, cu, su, ids, E, X.E4M3))
    assert X.near_codes(hidden.codes.cpu(), hidden.scales.cpu(), h, dh)
    for out in (torch.float32, torch.bfloat16):
        check(ops.fp8_moe_mm_ids(x, dev, g, E, u, out).view(T * n_used, mid), *X.gated(*by_pair(q, xs, cg, sg, ids, E, out), *by_pair(q, xs, cu, su, ids, E, out)))
        y, dy = by_pair(hidden.codes.cpu(), hidden.scales.cpu(), cd, sd, ids, E, out)
        check(ops.fp8_moe_mm_ids(hidden, dev, d, E, out_dtype=out).view(T * n_used, K), y, dy)


@pytest.mark.parametrize("T,n_used,E,mid,K,fused", [(1, 12, 16, 272, 144, True), (2, 9, 64, 48, 16, True), (3, 1, 8, 1040, 130 * 16, True), (1, 60, 64, 512, 64, True), (1, 400, 512, 512, 32, False),
                                                    (1, 2, 4, 8320, 32, False), (7, 2, 14, 64, 4112, True)])
def test_second_products_with_their_sum(ops, T, n_used, E, mid, K, fused):
    (cg, sg), (cu, su), (cd, sd) = X.matrix(mid, K, 23, E), X.matrix(mid, K, 24, E), X.matrix(K, mid, 25, E, True)
    g, u, d = weight(ops, cg, sg, E), weight(ops, cu, su, E), weight(ops, cd, sd, E)
    ids = ids_for(T, n_used, E, 26)
    x, _, _ = give(X.rows(T, K, 27, False), "bf16")
    hidden = ops.fp8_moe_mm_ids(x, ids.cuda(), g, E, u, X.E4M3)
    y, dy = by_pair(hidden.codes.cpu(), hidden.scales.cpu(), cd, sd, ids, E, torch.float32)
    rows = ops.fp8_moe_experts_rows(x, g, u, d, ids.cuda(), E)
    check(rows.view(T * n_used, K), y, dy)
    wts = torch.randn((T, n_used), generator=torch.Generator().manual_seed(28))  # (of either sign)
    for dtype in (torch.float32, torch.bfloat16):
        w = wts.to(dtype).double()[:, :, None]
        y3, d3 = y.view(T, n_used, K), dy.view(T, n_used, K)
        got = ops.fp8_moe_experts(x, g, u, d, wts.to(dtype).cuda(), ids.cuda(), E)
        assert ("k_fp8_down" in ops.last_kernel()) == fused, ops.last_kernel()
        check(got, (y3 * w).sum(1), (d3 * w.abs()).sum(1) + (y3 * w).abs().sum(1) * (n_used + 1) * 2.0 ** -24)


def layer(ops, seed=30):
    """(matrices of a small layer, their codes and scales on the CPU)"""
    shapes = {"qkv": (400, 512, 1), "o": (512, 256, 1), "gate": (256, 512, 1), "up": (256, 512, 1), "down": (512, 256, 1), "eg": (128, 512, 8), "eu": (128, 512, 8), "ed": (512, 128, 8)}
    host = {k: X.matrix(r, c, seed + i, n) for i, (k, (r, c, n)) in enumerate(shapes.items())}
    return {k: weight(ops, *host[k], shapes[k][2]) for k in shapes}, host


def run_layer(ops, w, h, ids, wts):
    """Norm, projection, projection, norm, a shared expert whose hidden rows stay in 8 bits, routed experts, norm with their weighted sum."""
    x = ops.add_rmsnorm_fp8(h)
    q = ops.fp8_linear(x, w["qkv"])
    o = ops.fp8_linear(q[:, :256], w["o"])
    x2, h2 = ops.add_rmsnorm_fp8(h, o, want_sum=True)
    hidden = ops.fp8_linear_glu2(x2, w["gate"], w["up"], X.E4M3)
    shared = ops.fp8_linear(hidden, w["down"])
    ys = ops.fp8_moe_experts_rows(x2, w["eg"], w["eu"], w["ed"], ids, 8)
    both = ops.fp8_moe_experts(x2, w["eg"], w["eu"], w["ed"], wts, ids, 8)
    x3, h3, n3 = ops.add_rmsnorm_fp8(h2, shared, ys=ys, topk_weights=wts, want_sum=True, want_norm=True)
    return x, q, o, x2, h2, hidden, shared, ys, both, x3, h3, n3


def flat(values):
    return [t for v in values for t in ((v.codes.view(torch.uint8), v.scales) if hasattr(v, "codes") else (v,))]


def inputs(T, seed):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn((T, 512), generator=g).to(torch.bfloat16)
    wts, ids = torch.softmax(torch.randn((T, 8), generator=g), 1).topk(3, 1)
    return h.cuda(), ids.cuda(), wts.cuda()


@pytest.mark.parametrize("T", [1, 7, 40, 300])
def test_a_layer(ops, T):
    """Every operator against 64 bits on what the one ahead of it left."""
    w, m = layer(ops)
    h, ids, wts = inputs(T, T)
    x, q, o, x2, h2, hidden, shared, ys, both, x3, h3, n3 = run_layer(ops, w, h, ids, wts)
    at = lambda r: (r.codes.cpu(), r.scales.cpu())  # noqa: E731
    norm = lambda v: v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-6)  # noqa: E731
    tiny = lambda v: v.abs() * 2.0 ** -23  # noqa: E731
    y = norm(h.cpu().double())
    assert X.near_codes(*at(x), y, tiny(y))
    check(q, *X.product(*at(x), *m["qkv"], torch.bfloat16))
    check(o, *X.product(*X.quantize(q[:, :256].cpu()), *m["o"], torch.bfloat16))
    y = h.cpu().double() + o.cpu().double()
    check(h2, y, tiny(y))
    assert X.near_codes(*at(x2), norm(y), tiny(norm(y)))
    assert X.near_codes(*at(hidden), *X.gated(*X.product(*at(x2), *m["gate"]), *X.product(*at(x2), *m["up"])))
    check(shared, *X.product(*at(hidden), *m["down"], torch.bfloat16))
    mids = ops.fp8_moe_mm_ids(x2, ids, w["eg"], 8, w["eu"], X.E4M3)
    e, de = by_pair(*at(mids), *m["ed"], ids.cpu(), 8)
    check(ys.view(T * 3, 512), e, de)
    wt = wts.cpu().double()[:, :, None]
    e, de = e.view(T, 3, 512), (de + (e.abs() + de) * BF16_HALF).view(T, 3, 512)
    check(both, (e * wt).sum(1), (de * wt).sum(1) + (e * wt).abs().sum(1) * 4 * 2.0 ** -24)
    y = h2.cpu().double() + shared.cpu().double() + (ys.cpu().double() * wt).sum(1)
    check(h3, y, tiny(y))
    check(n3, norm(y), tiny(norm(y)))
    assert X.near_codes(*at(x3), norm(y), tiny(norm(y)))


@pytest.mark.parametrize("T", [1, 40, 300])
def test_a_layer_captured(ops, T):
    """Two graphs with one memory pool, replayed in turn on new inputs with eager calls between them: the eager results bit for bit."""
    w, _ = layer(ops)
    state = [inputs(T, 50 + i) for i in range(2)]
    graphs, outs, pool = [], [], None
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in state:
            run_layer(ops, w, *s)
    torch.cuda.current_stream().wait_stream(side)
    for s in state:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            out = run_layer(ops, w, *s)
        pool = g.pool()
        graphs.append(g)
        outs.append(flat(out))
    for k in range(4):
        i = k % 2
        for t, new in zip(state[i], inputs(T, 60 + k)):
            t.copy_(new)
        graphs[i].replay()
        got = [t.clone() for t in outs[i]]  # (the other graph may use this one's memory)
        torch.cuda.synchronize()
        for a, b in zip(got, flat(run_layer(ops, w, *state[i])), strict=True):
            assert torch.equal(a, b)


def test_two_streams(ops):
    """The same weights from two streams at once, neither the default one."""
    w, _ = layer(ops)
    state = [inputs(T, 70 + T) for T in (1, 300)]
    want = [[t.clone() for t in flat(run_layer(ops, w, *s))] for s in state]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in state]
    for _ in range(3):
        got = []
        for s, st in zip(state, streams):
            with torch.cuda.stream(st):
                got.append([flat(run_layer(ops, w, *s)) for _ in range(4)])
        torch.cuda.synchronize()
        for runs, a in zip(got, want):
            for r in runs:
                assert all(torch.equal(p, q) for p, q in zip(r, a, strict=True))


@pytest.mark.parametrize("T", [0, 1, 7, 40, 300])
def test_native_calls_answer_as_the_others(ops, T, monkeypatch):
    """The calls' native way and the one through ctypes: the same results, and the same refusals."""
    w, _ = layer(ops)
    h, ids, wts = inputs(max(T, 1), T)
    h, ids, wts = h[:T], ids[:T], wts[:T]
    gamma = torch.rand(512, device="cuda").to(torch.bfloat16)

    def results():
        r = [*(run_layer(ops, w, h, ids, wts) if T else ())]
        rows = ops.fp8_quantize_rows(h)
        r += [ops.add_rmsnorm_fp8(h, h, h, gamma=gamma), *ops.add_rmsnorm_fp8(h, h, gamma=gamma, eps=0.5, want_norm=True), ops.fp8_linear(rows, w["qkv"]),
              ops.fp8_linear(h.float(), w["qkv"], out_dtype=torch.float32), ops.fp8_linear(h, w["qkv"], gamma[:400]), ops.fp8_linear_glu2(rows, w["gate"], w["up"]),
              ops.fp8_linear_glu2(h, w["gate"], w["up"], torch.float32), ops.fp8_moe_experts(h, w["eg"], w["eu"], w["ed"], wts.to(torch.bfloat16), ids.int(), 8),
              ops.fp8_moe_experts(rows, w["eg"], w["eu"], w["ed"], wts, ids, 8), ops.fp8_linear(h[None], w["qkv"])]
        return [t.clone() for t in flat(r)]

    def refusals():
        return (lambda: ops.add_rmsnorm_fp8(h.float()), lambda: ops.add_rmsnorm_fp8(h, h[:, :256]), lambda: ops.add_rmsnorm_fp8(h, gamma=gamma[:256]), lambda: ops.fp8_linear(h[:, :256], w["qkv"]),
                lambda: ops.fp8_linear(h.half(), w["qkv"]), lambda: ops.fp8_linear(h, w["eg"]), lambda: ops.fp8_linear(h, w["qkv"], out_dtype=torch.float16),
                lambda: ops.fp8_linear_glu2(h, w["gate"], w["qkv"]), lambda: ops.fp8_moe_experts(h, w["eg"], w["eu"], w["ed"], wts, ids, 7),
                lambda: ops.fp8_moe_experts(h, w["eg"], w["eu"], w["eu"], wts, ids, 8), lambda: ops.fp8_moe_experts(h, w["eg"], w["eu"], w["ed"], wts[:, :2], ids, 8),
                lambda: ops.fp8_moe_experts(h, w["eg"], w["eu"], w["ed"], wts, ids.float(), 8), lambda: ops.fp8_moe_experts(h, w["eg"], w["eu"], w["ed"], wts.cpu(), ids, 8))

    native = results()
    refused = []
    for call in refusals():
        with pytest.raises(ValueError):
            call()
        refused.append(True)
    monkeypatch.setattr(ops, "_host_calls", ops._NoNativeCalls)
    for a, b in zip(native, results(), strict=True):
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b)
    for call in refusals():
        with pytest.raises(ValueError):
            call()


def test_registered_operators(ops):
    from orin_qwen_lossless_amd import torch_ops  # noqa: F401

    B = torch.ops.bf16n
    w, _ = layer(ops)
    h, ids, wts = inputs(7, 80)
    m = lambda k: [w[k].codes, w[k].scales]  # noqa: E731
    rows, total = ops.add_rmsnorm_fp8(h, h, want_sum=True)
    got = B.add_rmsnorm_fp8(h, h, None, None, None, None, 1e-6)
    assert all(torch.equal(a.view(b.dtype), b) for a, b in zip(got, flat((rows, total))))
    assert all(torch.equal(a.view(b.dtype), b) for a, b in zip(B.fp8_quantize_rows(h), flat((ops.fp8_quantize_rows(h),))))
    assert torch.equal(B.fp8_linear(got[0], got[1], *m("qkv"), None, False), ops.fp8_linear(rows, w["qkv"], out_dtype=torch.float32))
    assert torch.equal(B.fp8_linear(h, None, *m("qkv"), None, True), ops.fp8_linear(h, w["qkv"]))
    assert torch.equal(B.fp8_linear_glu2(got[0], got[1], *m("gate"), *m("up"), True), ops.fp8_linear_glu2(rows, w["gate"], w["up"]))
    assert torch.equal(B.fp8_moe_experts(h, None, m("eg"), m("eu"), m("ed"), wts, ids, 8), ops.fp8_moe_experts(h, w["eg"], w["eu"], w["ed"], wts, ids, 8))


def test_scales_of_any_strides(ops):
    """Activations' scales by rows, by blocks, out of a wider table, and one scale for all of a row's blocks."""
    c, s = X.matrix(200, 512, 31)
    w = weight(ops, c, s)
    for T in (3, 40):
        q, xs = X.quantize(X.rows(T, 512, 32))
        wide = torch.full((2 * T, 9), float("nan"), device="cuda")
        wide[::2, 1::2] = xs.cuda()
        want = ops.fp8_linear(ops.Fp8Rows(q.cuda(), xs.cuda()), w)
        check(want, *X.product(q, xs, c, s, torch.bfloat16))
        for given in (xs.t().contiguous().cuda().t(), wide[::2, 1::2]):
            assert torch.equal(ops.fp8_linear(ops.Fp8Rows(q.cuda(), given), w), want)
        one = xs[:, :1].cuda().expand(T, 4)
        check(ops.fp8_linear(ops.Fp8Rows(q.cuda(), one), w), *X.product(q, one.cpu(), c, s, torch.bfloat16))


def test_codes_beyond_four_gigabytes(ops):
    """Places past 32 bits in the weights, for every kernel: the last rows of a large matrix are those of a small one."""
    rows, K = 280000, 16384
    big = torch.empty((rows, K), dtype=torch.uint8, device="cuda")
    big.random_(0, 0x78, generator=torch.Generator(device="cuda").manual_seed(33))
    s = torch.rand((-(-rows // 128), K // 128), generator=torch.Generator(device="cuda").manual_seed(34), device="cuda") * 1e-4
    c = big.view(X.E4M3)
    w = ops.Fp8Weight(c, s)
    tail = rows % 128 + 128
    tc, ts = c[-tail:].cpu(), s[-2:].cpu()
    for T in (1, 20, 40):
        q, xs = X.quantize(X.rows(T, K, 35, False))
        y, dy = X.product(q, xs, tc, ts, torch.bfloat16)
        check(ops.fp8_linear(ops.Fp8Rows(q.cuda(), xs.cuda()), w)[:, -tail:], y, dy)
    n = 2  # two matrices of 140000 rows: their last blocks are cut short
    stack = ops.Fp8Weight(c, torch.rand((n * -(-(rows // n) // 128), K // 128), device="cuda") * 1e-4, n)
    cut = rows // n % 128
    for T in (2, 40):
        ids = torch.full((T, 1), 1, dtype=torch.int32, device="cuda")
        q, xs = X.quantize(X.rows(T, K, 36, False))
        y, dy = X.product(q, xs, c[-cut:].cpu(), stack.scales[-1:].cpu(), torch.bfloat16)
        check(ops.fp8_moe_mm_ids(ops.Fp8Rows(q.cuda(), xs.cuda()), ids, stack, n, out_dtype=torch.bfloat16)[:, 0, -cut:], y, dy)


def test_rows_beyond_four_gigabytes(ops):
    """Activation rows and results so far apart that their places pass 32 bits."""
    c, s = X.matrix(200, 256, 37)
    w = weight(ops, c, s)
    for T in (20, 70):
        x, q, xs = give(X.rows(T, 256, 38), "bf16")
        far = torch.empty(T * (5 << 27), dtype=torch.uint8, device="cuda").view(torch.bfloat16).as_strided((T, 256), (5 << 26, 1))
        far.copy_(x)
        want = ops.fp8_linear(x, w)
        assert torch.equal(ops.fp8_linear(far, w), want)
        codes = torch.empty(T * (5 << 26), dtype=torch.uint8, device="cuda").as_strided((T, 256), (5 << 26, 1))
        codes.copy_(q.cuda().view(torch.uint8))
        assert torch.equal(ops.fp8_linear(ops.Fp8Rows(codes.view(X.E4M3), xs.cuda()), w), want)
        del far, codes
    # 2^32 results and more: the last token's are those of one token alone
    R, K, T = 1 << 20, 16, 4200
    c, s = X.matrix(R, K, 39)
    x, _, _ = give(X.rows(T, K, 40, False), "bf16")
    y = ops.fp8_linear(x, weight(ops, c, s))
    alone = ops.fp8_linear(x[-1:], weight(ops, c, s), out_dtype=torch.float32).cpu().double()
    _, dy = X.product(*X.quantize(x[-1:].cpu()), c, s, torch.bfloat16)
    check(y[-1:], alone, 2 * dy)


@pytest.mark.parametrize("T", [1, 5])
@pytest.mark.parametrize("dense", ["hybrid", "fp8"])
def test_decode_step_in_8_bits(ops, T, dense):
    """A layer of the decode step with such experts (and projections): the router's choice and the experts' rows from its own input, and the step as
    a graph against the eager one."""
    from orin_qwen_lossless_amd import decode_step as D
    from orin_qwen_lossless_amd import synth

    seed = [9000]

    def gen(rows, k):
        seed[0] += 1
        return synth.weights_torch(rows, k, seed[0], "cuda")

    sets, raw, nbytes = D.make_layer_sets(ops, gen, 1, True, "fp8", dense)
    w = sets[0]
    assert isinstance(w["gate"], ops.Fp8Weight) and nbytes["gate"] == w["gate"].nbytes and isinstance(w["qkv"], ops.Fp8Weight) == (dense == "fp8")
    head = ops.fp8_quantize(gen(512, D.K_MODEL))
    step = D.Bf16nStep(ops, sets, head, 2, T)
    x2 = torch.randn((T, D.K_MODEL), generator=torch.Generator().manual_seed(98)).to(torch.bfloat16).cuda()
    ys, wts, ids = step.experts(w, x2)
    v, i = ops.router_topk(ops.mmv(x2, w["router"]), D.TOPK)
    assert torch.equal(ids[:, :D.TOPK], i) and torch.equal(wts[:, :D.TOPK], v) and (ids[:, D.TOPK] == D.E).all()
    q, xs = X.quantize(x2.cpu())
    hidden = ops.fp8_moe_mm_ids(x2, ids, w["gate"], D.EA, w["up"], X.E4M3)
    cut = lambda m, e, n: (m.codes[e * n: e * n + n].cpu(), m.scales[e * (n // 128): (e + 1) * (n // 128)].cpu())  # noqa: E731
    for t in range(T):
        for j in (0, D.TOPK):
            e, p = int(ids[t, j]), t * (D.TOPK + 1) + j
            h = X.gated(*X.product(q[t: t + 1], xs[t: t + 1], *cut(w["gate"], e, D.N_MID)), *X.product(q[t: t + 1], xs[t: t + 1], *cut(w["up"], e, D.N_MID)))
            hq, hs = hidden.codes[p: p + 1].cpu(), hidden.scales[p: p + 1].cpu()
            assert X.near_codes(hq, hs, *h)
            check(ys[t: t + 1, j], *X.product(hq, hs, *cut(w["down"], e, D.K_MODEL)))
    # a matrix in 8 bits is the exact one within half a step of its codes and of its block's smallest number
    back = X.weight64(w["gate"].codes.cpu(), w["gate"].scales.cpu(), D.EA)[3]
    exact = raw[0]["gate"][3 * D.N_MID: 4 * D.N_MID].double().cpu()
    most = w["gate"].scales.view(D.EA, -1, D.K_MODEL // 128)[3].double().cpu().repeat_interleave(128, 0).repeat_interleave(128, 1)
    assert ((back - exact).abs() <= exact.abs() * 2.0 ** -4 * (1 + 2.0 ** -20) + most * 2.0 ** -10).all()
    h = torch.randn((T, D.K_MODEL), generator=torch.Generator().manual_seed(99)).to(torch.bfloat16).cuda()
    graph, out = D.capture(step, h)
    for k in range(3):
        h.copy_(torch.randn((T, D.K_MODEL), generator=torch.Generator().manual_seed(100 + k)).to(torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step(h)) and out.shape == (T, 512)
    # without an output projection the step ends in the norm as BF16 numbers
    assert D.Bf16nStep(ops, sets, None, 1, T)(h).dtype is torch.bfloat16


@pytest.mark.parametrize("T,n_used,E,N,K", [(90, 2, 3, 384, 272), (70, 3, 4, 256, 4400), (200, 1, 2, 1024, 144), (65, 2, 5, 640, 9104)])
def test_lists_by_row_tiles(ops, T, n_used, E, N, K):
    """Two row tiles to a block: an odd number of them, a last block of columns that is cut, more steps than a register's lanes have scales."""
    (c, s), (cu, su) = X.matrix(N, K, 41, E, True), X.matrix(N, K, 42, E, True)
    ids = ids_for(T, n_used, E, 43)
    x, q, xs = give(X.rows(T, K, 44, False), "rows")
    for out in (torch.bfloat16, torch.float32):
        check(ops.fp8_moe_mm_ids(x, ids.cuda(), weight(ops, c, s, E), E, out_dtype=out).view(T * n_used, N), *by_pair(q, xs, c, s, ids, E, out))
        y, dy = X.gated(*by_pair(q, xs, c, s, ids, E, out), *by_pair(q, xs, cu, su, ids, E, out))
        check(ops.fp8_moe_mm_ids(x, ids.cuda(), weight(ops, c, s, E), E, weight(ops, cu, su, E), out).view(T * n_used, N), y, dy)


def test_more_lists_than_a_wavefront_finds_at_once(ops):
    """1200 matrices: lists are looked for 512 at a time."""
    E, N, K, T = 1200, 16, 32, 700
    c, s = X.matrix(N, K, 45, E)
    ids = torch.randint(-1, E + 1, (T, 2), generator=torch.Generator().manual_seed(46))
    ids[:200, 0] = E - 1
    x, q, xs = give(X.rows(T, K, 47, False), "f32")
    for out in (torch.bfloat16, torch.float32):
        check(ops.fp8_moe_mm_ids(x, ids.cuda(), weight(ops, c, s, E), E, out_dtype=out).view(2 * T, N), *by_pair(q, xs, c, s, ids, E, out))
