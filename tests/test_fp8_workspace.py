"""8-bit floating point with block scales: the workspaces that the C calls ask for, without a GPU."""
from __future__ import annotations

import ctypes as C

import pytest

from orin_qwen_lossless_amd import _lib

CODES, BF16, F32 = 0, 1, 2


def weight(rows, K, n=1):
    return _lib.Fp8Weight(4096, 4096, K, rows, n, 0, 0)


def product_bytes(w, up, x_kind, y_kind, x_rows, n_pairs=0, listed=0):
    n = C.c_uint64(1 << 63)
    _lib.check(_lib.lib().bf16n_fp8_workspace_bytes(C.byref(w), up, x_kind, y_kind, x_rows, n_pairs, listed, C.byref(n)))
    return n.value


@pytest.mark.parametrize("x_kind", [CODES, BF16, F32])
@pytest.mark.parametrize("y_kind", [CODES, BF16, F32])
def test_an_empty_batch_needs_none(x_kind, y_kind):
    for w in (weight(1408, 2048), weight(0, 2048), weight(16, 16), weight(4 * 256, 128, 4)):
        for listed in (0, 1):
            assert product_bytes(w, int(y_kind == CODES), x_kind, y_kind, 0, 0, listed) == 0


COUNTS = [*range(1, 200), 255, 256, 300, 511, 512, 513, 1000, 2048, 4096, 8191, 8192, 8193, 20000]


@pytest.mark.parametrize("rows,K", [(1408, 2048), (512, 2048), (16, 16), (16, 1040), (48, 32768), (8192, 8192), (8208, 512), (144, 900 * 16), (1 << 20, 128)])
@pytest.mark.parametrize("x_kind", [CODES, BF16, F32])
@pytest.mark.parametrize("up,y_kind", [(0, BF16), (0, F32), (1, BF16), (1, CODES)])
def test_the_size_for_many_tokens_is_enough_for_fewer(rows, K, x_kind, up, y_kind):
    sizes = [product_bytes(weight(rows, K), up, x_kind, y_kind, n) for n in COUNTS]
    assert sizes == sorted(sizes)


@pytest.mark.parametrize("E,mid,K,n_used", [(256, 512, 2048, 8), (8, 1408, 2048, 2), (4, 48, 64, 3), (64, 8320, 32, 1), (512, 512, 32, 400), (1, 16, 16, 1)])
@pytest.mark.parametrize("x_kind", [CODES, BF16, F32])
@pytest.mark.parametrize("weighted", [0, 1])
def test_the_same_of_the_experts(E, mid, K, n_used, x_kind, weighted):
    gate, down, n, sizes = weight(E * mid, K, E), weight(E * K, mid, E), C.c_uint64(), []
    for tokens in COUNTS:
        _lib.check(_lib.lib().bf16n_fp8_moe_experts_workspace_bytes(C.byref(gate), C.byref(down), x_kind, weighted, tokens, n_used, C.byref(n)))
        sizes.append(n.value)
    assert sizes == sorted(sizes)


def test_sizes_and_kinds_that_the_calls_refuse():
    """No size for them either: 2^62 rows passed 64 bits and came back as none."""
    L, n, w = _lib.lib(), C.c_uint64(), weight(4 * 128, 256, 4)
    ask = lambda *a: L.bf16n_fp8_workspace_bytes(C.byref(w), *a, C.byref(n))  # noqa: E731
    assert ask(1, BF16, CODES, 1 << 28, 1 << 28, 0) == 0 and n.value == (1 << 28) * 128 * 4  # (the blocks make the codes of so short rows)
    for bad in ((0, BF16, BF16, (1 << 28) + 1, 0, 0), (0, BF16, BF16, 1 << 62, 0, 0), (0, CODES, BF16, 1, 1 << 62, 1), (0, 3, BF16, 1, 0, 0), (0, -1, BF16, 1, 0, 0), (0, CODES, 3, 1, 0, 0)):
        assert ask(*bad) == _lib.EINVAL and L.bf16n_last_error().startswith(b"bf16n: fp8"), bad
    down = weight(1024, 128, 4)
    for kind in (-1, 3):
        assert L.bf16n_fp8_moe_experts_workspace_bytes(C.byref(w), C.byref(down), kind, 1, 10, 2, C.byref(n)) == _lib.EINVAL
