"""Rules of the products of microscaled operands on the host: sizes at their ends, and which kernel a call takes (nothing is launched)."""
import ctypes as C
import os
import subprocess
import sys
from pathlib import Path

import pytest

from test_mx_scaled_plans_gpu import KIND, TILES
from tyloquant_amd import _lib as L


@pytest.fixture(scope="module")
def lib():
    lib = L.lib()
    lib.mfq_hip_set_cu_count(256)
    yield lib
    lib.mfq_hip_set_cu_count(0)


@pytest.mark.parametrize("act", [4, 6])
@pytest.mark.parametrize("x_quantized", [0, 1])
def test_sizes_of_the_longest_rows(lib, act, x_quantized):
    """Rows of up to 2^31 - 32 columns: as many whole groups of 256 as 2^31 columns have."""
    first, last = (1 << 31) - 224, (1 << 31) - 32      # of the last group
    assert lib.mfq_hip_mx_scale_bytes(3, first) == lib.mfq_hip_mx_scale_bytes(3, last) == 1 << 31
    assert lib.mfq_hip_mx_quantized_row_bytes(act, first) == lib.mfq_hip_mx_quantized_row_bytes(act, last) == (1 << 23) * (128 if act == 4 else 192)
    # 40 rows: the pieces of K, as many for a group fewer, and those rows quantised, which that group's codes and scales make longer
    fewer, *need = [lib.mfq_hip_mx_scaled_gemm_workspace_bytes(act, 64, k, 40, x_quantized) for k in (first - 32, first, last)]
    assert [n - fewer for n in need] == [0 if x_quantized else 40 * (128 if act == 4 else 192) + 2 * 256] * 2


@pytest.mark.parametrize("act,cus,rows,out,K,plan,pieces", TILES)
def test_tile_of_a_call(lib, act, cus, rows, out, K, plan, pieces):
    lib.mfq_hip_set_cu_count(cus)
    try:
        got = C.c_int()
        assert (lib.mfq_hip_mx_scaled_plan(KIND[act], out, K, rows, 0, C.byref(got)), got.value) == (plan, pieces)
    finally:
        lib.mfq_hip_set_cu_count(256)


def test_every_tile_is_run():
    """By the tests on the card, whole and with K in pieces (of 256 x 128 MXFP4 no call was found that splits K)."""
    assert {(plan, pieces > 1) for *_, plan, pieces in TILES} == {(p, s) for p in range(5, 13) for s in (False, True)} - {(8, True)}


@pytest.mark.parametrize("act,out,K,rows,glu,plan", [
    (4, 12288, 4096, 1, 0, 0), (4, 12288, 4096, 16, 0, 0), (4, 12288, 4096, 17, 0, 2), (4, 12288, 4096, 33, 0, 6), (4, 12288, 4096, 601, 0, 7),
    (4, 17408, 5120, 8192, 0, 9), (6, 24576, 4096, 2048, 1, 11), (6, 4096, 12288, 13, 0, 3), (6, 4096, 12288, 4, 0, 0),
    (6, 96, 5632, 20, 0, 2), (6, 96, 5632, 20, 1, 4), (4, 96, 8224, 20, 0, 2), (4, 96, 8224, 20, 1, 4), (4, 96, 17440, 5, 1, 3), (4, 96, 17440, 16, 0, 3),
    (4, 64, 48, 1, 0, -1), (5, 64, 64, 1, 0, -1), (4, 0, 64, 1, 0, -1), (4, 64, 64, 0, 0, -1), (4, 64, (1 << 24) + 32, 40, 0, -1)])
def test_kernel_of_a_call(lib, act, out, K, rows, glu, plan):
    assert lib.mfq_hip_mx_scaled_plan(act, out, K, rows, glu, None) == plan


@pytest.mark.parametrize("act,K,pairs,E,mapped,glu,x_quantized,plan", [
    (6, 4096, 8, 64, 0, 1, 0, 0), (4, 2048, 488, 64, 1, 0, 0, 0), (4, 2048, 488, 64, 1, 0, 1, 1), (4, 4128, 60, 16, 1, 0, 0, 1),
    (4, 2048, 640, 64, 1, 0, 0, 0), (4, 2048, 641, 64, 1, 0, 0, 5), (6, 2048, 641, 64, 1, 0, 0, 10),       # ten pairs an expert
    (4, 2048, 64 * 159, 64, 1, 0, 0, 5), (4, 2048, 64 * 159 + 1, 64, 1, 0, 0, 8), (6, 1440, 6004, 32, 1, 0, 0, 11),
    (4, 17440, 24, 8, 1, 0, 0, 3), (6, 12288, 24, 8, 1, 1, 1, 3), (4, 15136, 24, 8, 1, 0, 0, 1), (4, 15136, 24, 8, 1, 1, 0, 3),
    (8, 64, 1, 1, 1, 0, 0, -1), (4, 40, 1, 1, 1, 0, 0, -1), (4, 64, 0, 1, 1, 0, 0, -1)])
def test_kernel_of_routed_experts(lib, act, K, pairs, E, mapped, glu, x_quantized, plan):
    assert lib.mfq_hip_mx_moe_plan(act, K, pairs, E, mapped, glu, x_quantized) == plan


@pytest.mark.parametrize("act", [4, 6])
@pytest.mark.parametrize("out", [300, 301, 302, 303, 304, 134, 32])
def test_partial_sums_begin_on_16_bytes(lib, act, out):
    """K in pieces: a row of partial sums has two halves, gate and up of a gated call, that 16-byte stores fill from their first column on."""
    pieces, rows, K = C.c_int(), 64, 4096
    assert lib.mfq_hip_mx_scaled_plan(act, out, K, rows, 0, C.byref(pieces)) >= 5 and pieces.value > 1
    half, left = divmod(lib.mfq_hip_mx_scaled_gemm_workspace_bytes(act, out, K, rows, 1), pieces.value * rows * 2)
    assert left == 0 and half % 16 == 0 and half >= -(-out // 2) * 4


def _plans_with(env):
    """plans in a process that starts with these knobs: MXFP4 and MXFP6 of 12288 x 4096 at 601 rows and of 64 x 64 at 40, experts with 3, 30 and 300
    pairs each"""
    code = ("import ctypes as C\nfrom tyloquant_amd import _lib as L\nl, n = L.lib(), C.c_int()\nl.mfq_hip_set_cu_count(256)\n"
            "for a in (4, 6):\n    for out, K, M in ((12288, 4096, 601), (64, 64, 40)):\n"
            "        print(l.mfq_hip_mx_scaled_plan(a, out, K, M, 0, C.byref(n)), n.value)\n"
            "    print(*[l.mfq_hip_mx_moe_plan(a, 2048, 8 * p, 8, 1, 0, 1) for p in (3, 30, 300)])\n")
    root = Path(__file__).resolve().parents[1]
    out = subprocess.run([sys.executable, "-c", code], env={**os.environ, "PYTHONPATH": str(root), **env}, check=True, capture_output=True, text=True).stdout
    return [[int(v) for v in line.split()] for line in out.splitlines()]


def test_knobs_mean_one_thing():
    """A tile is heeded by the calls of its kind and no other, pieces where K has as many groups, the experts' kernel by experts alone."""
    plain = _plans_with({})
    assert plain[2] == [1, 5, 8] and plain[5] == [1, 10, 11]
    tile = _plans_with({"MFQ_MXS_TILE": "2"})       # 64 x 128 of MXFP4
    assert tile[0][0] == tile[1][0] == 6 and tile[2:] == plain[2:]
    tile = _plans_with({"MFQ_MXS_TILE": "8"})       # 256 x 192 of MXFP6
    assert tile[3][0] == tile[4][0] == 12 and tile[:3] == plain[:3] and tile[5] == plain[5]
    assert _plans_with({"MFQ_MXS_TILE": "9"}) == plain and _plans_with({"MFQ_MXS_SPLIT": "17"}) == plain
    pieces = _plans_with({"MFQ_MXS_SPLIT": "4"})
    assert [pieces[i][1] for i in (0, 3)] == [4, 4] and [pieces[i] for i in (1, 2, 4, 5)] == [plain[i] for i in (1, 2, 4, 5)]
    experts = _plans_with({"MFQ_MXS_EXPERTS": "2"})
    assert experts[2] == [5, 5, 5] and experts[5] == [10, 10, 10] and [experts[i] for i in (0, 1, 3, 4)] == [plain[i] for i in (0, 1, 3, 4)]
