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
