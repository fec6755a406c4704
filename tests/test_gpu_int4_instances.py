"""Every instance of the products' kernels on 4-bit weights with group scales, against the definition in 64 bits (int4_exact: the bounds
are derived there), at shapes whose rows, columns and K end inside a tile.  Each test says which instance it is about and fails if the
call went to another, so that a changed rule cannot leave one untested."""
from __future__ import annotations

import pytest
import torch

import int4_exact as X
from test_gpu_int4 import acts, weight

pytestmark = pytest.mark.gpu

GROUP_CLASS = {32: 2, 64: 1, 128: 0, 256: 0, 512: 0}  # the template argument for a group's size


def text(v):
    return str(v).lower() if isinstance(v, bool) else str(v)


def instance(name, *args):
    return f"{name}<{', '.join(map(text, args))}>"


@pytest.mark.parametrize("glu", [False, True])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype,T,tiles", [(torch.bfloat16, 5, 1), (torch.bfloat16, 21, 2), (torch.float32, 6, 1)])
@pytest.mark.parametrize("kernel,rows,K", [("k_i4_small", 300, 1312), ("k_i4_few", 8250, 1312)])
def test_few_columns(ops, kernel, rows, K, dtype, T, tiles, group, zeros, glu):
    w, dw = weight(ops, rows, K, group, 400, zeros)
    x = acts(T, K, 401, dtype)
    y, b = X.product(x, w)
    f32, gm = dtype is torch.float32, GROUP_CLASS[group]
    if glu:
        w2, dw2 = weight(ops, rows, K, group, 402, zeros, True)
        y, b = X.gated(y, b, *X.product(x, w2))
        got = ops.int4_mmv_glu2(x.cuda(), dw, dw2)
    else:
        got = ops.int4_mmv(x.cuda(), dw)
    args = (tiles, gm, glu, f32, zeros) if kernel == "k_i4_small" else (tiles, 2 if glu else 1, gm, glu, f32, zeros, 8)
    assert ops.last_kernel() == instance(kernel, *args)
    X.check(got, y, b)


@pytest.mark.parametrize("glu", [False, True])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True), (512, False)])
@pytest.mark.parametrize("cols,rows,K,T", [(64, 4100, 1056, 200), (64, 8330, 416, 70), (64, 2050, 544, 3000), (128, 4100, 288, 4101), (128, 33000, 160, 529)])
def test_many_columns(ops, cols, rows, K, T, group, zeros, glu):
    """Tiles of 128 x 64 and 128 x 128, gated ones of 64 rows of either matrix."""
    w, dw = weight(ops, rows, K, group, 410, zeros)
    x = acts(T, K, 411)
    y, b = X.product(x, w)
    dw2 = None
    if glu:
        w2, dw2 = weight(ops, rows, K, group, 412, zeros, True)
        y, b = X.gated(y, b, *X.product(x, w2))
    for out in (torch.float32, torch.bfloat16):
        got = ops.int4_mmv_glu2(x.cuda(), dw, dw2, out_dtype=out) if glu else ops.int4_mmv(x.cuda(), dw, out_dtype=out)
        shape = (2, 2, 4, 4) if cols == 128 else (1, 4, 4, 2)
        assert ops.last_kernel() == instance("k_i4_many", *shape, GROUP_CLASS[group], glu, False)
        X.check(got, y, X.rounded(y, b, out), out)


def ids_of(counts, n_used, E, seed):
    """ids [tokens, n_used] that name expert e counts[e] times, in no order; the rest of the last token, and five more, name none"""
    flat = torch.repeat_interleave(torch.arange(E), torch.tensor(counts))
    none = 5 + (-(len(flat) + 5)) % n_used
    flat = torch.cat([flat, torch.tensor([-1, E, E + 7, -5, 1 << 20] + [-1] * (none - 5))])
    return flat[torch.randperm(len(flat), generator=torch.Generator().manual_seed(seed))].view(-1, n_used).to(torch.int32)


def check_lists(ops, kernel, E, N, K, group, zeros, counts, n_used, glu, dtypes=(torch.float32, torch.bfloat16)):
    w, dw = weight(ops, E * N, K, group, 420, zeros)
    w2, dw2 = weight(ops, E * N, K, group, 421, zeros, True)
    ids = ids_of(counts, n_used, E, 422)
    T = ids.shape[0]
    cut = lambda m, e: (*(None if p is None else p[e * N: e * N + N] for p in m[:3]), group)  # noqa: E731
    for x in (acts(T, K, 423), acts(T * n_used, K, 424).view(T, n_used, K)):
        xp = (x[:, None].expand(T, n_used, K) if x.dim() == 2 else x).reshape(-1, K)
        got = {}
        for out in dtypes:
            got[out] = ops.int4_moe_mm_ids(x.cuda(), ids.cuda(), dw, E, up=dw2 if glu else None, out_dtype=out).reshape(-1, N).cpu()
            assert ops.last_kernel() == kernel
        for e in range(E):
            at = (ids.reshape(-1) == e).nonzero()[:, 0]
            assert len(at) == counts[e]
            if len(at):
                y, b = X.product(xp[at], cut(w, e))
                if glu:
                    y, b = X.gated(y, b, *X.product(xp[at], cut(w2, e)))
                for out in dtypes:
                    X.check(got[out][at], y, X.rounded(y, b, out), (e, len(at), out))
        none = ((ids < 0) | (ids >= E)).reshape(-1)
        assert all(not g[none].any() for g in got.values())


@pytest.mark.parametrize("glu", [False, True])
@pytest.mark.parametrize("K,group,zeros", [(416, 32, True), (544, 32, False), (352, 64, False), (1056, 64, True), (160, 128, True), (544, 256, False)])
def test_lists_of_many_columns(ops, K, group, zeros, glu):
    """Pieces of every number of tiles of 16 columns, whole and cut short, of rows that end inside a tile."""
    counts = [1, 16, 17, 32, 33, 48, 49, 64, 65, 81, 97, 113, 0, 128, 130, 2]
    check_lists(ops, instance("k_i4_many", 1, 4, 4, 2, GROUP_CLASS[group], glu, True), 16, 165, K, group, zeros, counts, 8, glu)


@pytest.mark.parametrize("glu", [False, True])
@pytest.mark.parametrize("K,group,zeros", [(416, 32, False), (352, 64, True), (288, 128, False)])
def test_lists_of_one_expert_and_of_many(ops, K, group, zeros, glu):
    """All columns with one expert; more experts than a round of the pieces' table has, most of them with nothing."""
    check_lists(ops, instance("k_i4_many", 1, 4, 4, 2, GROUP_CLASS[group], glu, True), 1, 130, K, group, zeros, [200], 3, glu, (torch.float32,))
    counts = [0] * 300
    counts[0], counts[255], counts[256], counts[299] = 1500, 70, 2100, 33
    check_lists(ops, instance("k_i4_many", 1, 4, 4, 2, GROUP_CLASS[group], glu, True), 300, 20, K, group, zeros, counts, 2, glu, (torch.float32,))


@pytest.mark.parametrize("glu", [False, True])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("kernel,N,K,share", [("k_i4_few", 330, 352, 0), ("k_i4_few", 330, 352, 1), ("k_i4_few", 330, 352, 4), ("k_i4_few", 330, 1312, 9), ("k_i4_small", 37, 352, 4)])
def test_lists_of_few_columns(ops, kernel, N, K, share, group, zeros, glu):
    """Lists of `share` columns about, one of them longer than two passes, some empty."""
    E = 40
    counts = [share] * E
    counts[3], counts[7], counts[11], counts[39] = 37, 0, 1, share + 2
    gm = GROUP_CLASS[group]
    args = (1, gm, glu, False, zeros) if kernel == "k_i4_small" else (1, 2 if glu else 1, gm, glu, False, zeros, 8)
    check_lists(ops, instance(kernel, *args), E, N, K, group, zeros, counts, 3, glu, (torch.float32,))


@pytest.mark.parametrize("glu", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
@pytest.mark.parametrize("kernel,N", [("k_i4_few", 1045), ("k_i4_small", 45)])
def test_columns_by_ids(ops, kernel, N, group, zeros, dtype, glu):
    """A column to a (token, slot) pair, one activation row to a token or to a pair."""
    E, K, T, n_used = 6, 352, 4, 3
    w, dw = weight(ops, E * N, K, group, 430, zeros)
    w2, dw2 = weight(ops, E * N, K, group, 431, zeros, True)
    ids = torch.tensor([[0, 5, 5], [-1, 2, 6], [3, 3, 3], [1, 4, 0]], dtype=torch.int32)
    cut = lambda m, e: (*(None if p is None else p[e * N: e * N + N] for p in m[:3]), group)  # noqa: E731
    gm, f32 = GROUP_CLASS[group], dtype is torch.float32
    args = (1, gm, glu, f32, zeros) if kernel == "k_i4_small" else (1, 2 if glu else 1, gm, glu, f32, zeros, 8)
    for x in (acts(T, K, 432, dtype), acts(T * n_used, K, 433, dtype).view(T, n_used, K)):
        got = ops.int4_mmv_glu2(x.cuda(), dw, dw2, ids.cuda(), N) if glu else ops.int4_mmv(x.cuda(), dw, ids.cuda(), N)
        assert ops.last_kernel() == instance(kernel, *args)
        for t in range(T):
            for i in range(n_used):
                e = int(ids[t, i])
                if not 0 <= e < E:
                    assert not got[t, i].any()
                    continue
                xi = (x[t] if x.dim() == 2 else x[t, i])[None]
                y, b = X.product(xi, cut(w, e))
                if glu:
                    y, b = X.gated(y, b, *X.product(xi, cut(w2, e)))
                X.check(got[t, i: i + 1], y, b, (t, i))


def test_activation_rows_too_far_apart_for_the_kernel_of_many_columns(ops):
    """Its places of activations are 32 bits: a product that it would take otherwise goes to the kernels for few, dense and by lists."""
    import ctypes as C

    from orin_qwen_lossless_amd import _lib

    w, dw = weight(ops, 8300, 416, 32, 440)
    x = acts(70, 416, 441)
    y, b = X.product(x, w)
    X.check(ops.int4_mmv(x.cuda(), dw), y, b)
    assert ops.last_kernel().startswith("k_i4_many<")
    space = torch.empty(70 * 35_000_000, dtype=torch.bfloat16, device="cuda")
    far = space.as_strided((70, 416), (35_000_000, 1))
    far.copy_(x)
    X.check(ops.int4_mmv(far, dw), y, b)
    assert ops.last_kernel().startswith(("k_i4_few<", "k_i4_small<"))

    E, N, K, T = 2, 165, 160, 40
    w, dw = weight(ops, E * N, K, 64, 442)
    x = acts(T, K, 443)
    ids = ids_of([25, 10], 1, E, 444)
    pairs, bounds = ops.int4_route(ids.cuda(), E)
    cw, out = ops._c_int4(dw), {}
    for apart in (K, 60_000_000):
        rows = space.as_strided((T, K), (apart, 1))
        rows.copy_(x)
        got = torch.empty((T, N), device="cuda")
        ws = ops._int4_workspace(cw, T, got.device, T, E)
        _lib.check(_lib.lib().bf16n_int4_mm_ids(C.byref(cw), None, rows.data_ptr(), apart, 0, pairs.data_ptr(), bounds.data_ptr(), got.data_ptr(), 0, N, E, T, 1,
                                                ws.data_ptr(), ws.numel(), ops._stream()))
        assert ops.last_kernel().startswith("k_i4_many<") == (apart == K)
        for t in range(T):
            e = int(ids[t, 0])
            if 0 <= e < E:
                y, b = X.product(x[t: t + 1], (*(p[e * N: e * N + N] for p in w[:3]), 64))
                X.check(got[t: t + 1], y, b, (apart, t))
            else:
                assert not got[t].any()
