"""The second products of few tokens: results are stored four at a time, at 16-byte aligned places of LDS, for every number of slots and blocks of K."""
from __future__ import annotations

import os
import shutil
import subprocess

import pytest
import torch

import fp8_exact as X
from test_gpu_fp8 import check, give, weight
from test_gpu_fp8_experts import by_pair, ids_for

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("g++") is None, reason="no g++")
def test_parts_are_aligned(tmp_path):
    exe = str(tmp_path / "layout")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=undefined", "-I" + os.path.join(ROOT, "orin_qwen_lossless_amd", "csrc"),
                    os.path.join(ROOT, "tests", "cpp", "fp8_down_layout.cpp"), "-o", exe], check=True, capture_output=True, timeout=120)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout


@pytest.mark.gpu
@pytest.mark.parametrize("T,n_used,mid", [(1, 1, 16), (2, 1, 720), (3, 2, 144), (1, 2, 1408), (2, 6, 1408), (4, 3, 272), (1, 5, 640), (1, 9, 912), (2, 10, 48)])
def test_slots_and_blocks_of_every_remainder(ops, T, n_used, mid):
    """slots * blocks of 1, 2 and 3 beyond a multiple of four"""
    E, K, out = 64, 64, 130
    (cg, sg), (cu, su), (cd, sd) = X.matrix(mid, K, 81, E), X.matrix(mid, K, 82, E), X.matrix(out, mid, 83, E)
    g, u, d = weight(ops, cg, sg, E), weight(ops, cu, su, E), weight(ops, cd, sd, E)
    ids = ids_for(T, n_used, E, 84)
    x, _, _ = give(X.rows(T, K, 85, False), "bf16")
    hidden = ops.fp8_moe_mm_ids(x, ids.cuda(), g, E, u, X.E4M3)
    y, dy = by_pair(hidden.codes.cpu(), hidden.scales.cpu(), cd, sd, ids, E, torch.float32)
    wts = torch.randn((T, n_used), generator=torch.Generator().manual_seed(86))
    w = wts.double()[:, :, None]
    y3, d3 = y.view(T, n_used, out), dy.view(T, n_used, out)
    got = ops.fp8_moe_experts(x, g, u, d, wts.cuda(), ids.cuda(), E)
    assert "k_fp8_down" in ops.last_kernel(), ops.last_kernel()
    check(got, (y3 * w).sum(1), (d3 * w.abs()).sum(1) + (y3 * w).abs().sum(1) * (n_used + 1) * 2.0 ** -24)
