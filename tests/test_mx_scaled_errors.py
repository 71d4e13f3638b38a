"""Products of microscaled operands without a GPU: argument checks of the C ABI (every rejected call launches nothing and leaves its
message), sizes, and the oracle's quantiser against closed forms."""
import ctypes as C

import numpy as np
import pytest
import torch

import mx_scaled_ref as P
from tyloquant_amd import _lib as L
from tyloquant_amd import formats as F
from tyloquant_amd.runtime_mx import MxWeight, mx_scaled_matmul

A = C.c_void_p(0x1000)      # an aligned address that a rejected call never dereferences
ODD = C.c_void_p(0x1001)


@pytest.fixture(scope="module")
def lib():
    return L.lib()


def _msg(lib):
    return lib.mfq_hip_last_error().decode()


def test_sizes(lib):
    assert [lib.mfq_hip_mx_quantized_row_bytes(4, k) for k in (32, 256, 288, 4096)] == [128, 128, 256, 2048]
    assert [lib.mfq_hip_mx_quantized_row_bytes(6, k) for k in (32, 256, 288, 2048)] == [192, 192, 384, 1536]
    assert lib.mfq_hip_mx_quantized_row_bytes(8, 256) == 0 and lib.mfq_hip_mx_quantized_row_bytes(4, 40) == 0
    assert [lib.mfq_hip_mx_scale_bytes(r, 288) for r in (1, 32, 33)] == [512, 512, 1024] and lib.mfq_hip_mx_scale_bytes(0, 256) == 0
    # a workspace that grows with the rows; none for rows that the kernel quantises itself or that come quantised
    assert lib.mfq_hip_mx_scaled_gemm_workspace_bytes(4, 4096, 4096, 1, 0) == 0
    assert lib.mfq_hip_mx_scaled_gemm_workspace_bytes(4, 4096, 4096, 16, 1) == 0
    assert lib.mfq_hip_mx_scaled_gemm_workspace_bytes(4, 4096, 8192, 16, 0) == 16 * 4096 + 32 * 256
    assert lib.mfq_hip_mx_scaled_gemm_workspace_bytes(4, 4096, 4096, 16, 0) == 0 and lib.mfq_hip_mx_scaled_gemm_workspace_bytes(4, 4096, 4096, 17, 0) > 0
    assert lib.mfq_hip_mx_scaled_gemm_workspace_bytes(5, 4096, 4096, 16, 0) == 0
    # routed experts: the rows and, where tiles serve the call, 16 bytes for each of at most so many and one
    moe = lib.mfq_hip_mx_moe_workspace_bytes
    assert moe(6, 8192, 100, 200, 64, 1, 0) == 100 * 6144 + 128 * 256 and moe(6, 8192, 100, 200, 64, 1, 1) == 0 and moe(6, 4096, 100, 200, 64, 1, 0) == 0
    assert moe(6, 288, 100, 1600, 32, 1, 1) == 16 * (25 + 32 + 1) and moe(6, 288, 100, 1600, 32, 1, 0) == 100 * 384 + 128 * 16 + 16 * 58
    assert moe(6, 288, 100, 200, 64, 0, 0) == 0


def test_quantize_checks(lib):
    q = lib.mfq_hip_mx_quantize_rows
    assert q(4, None, L.X_BF16, 256, 1, 256, A, A, None) == L.ERR_INVALID
    assert q(8, A, L.X_BF16, 256, 1, 256, A, A, None) == L.ERR_INVALID and "kind=8" in _msg(lib)
    assert q(4, A, 7, 256, 1, 256, A, A, None) == L.ERR_INVALID and "x_dtype" in _msg(lib)
    assert q(4, A, L.X_BF16, 256, 1, 250, A, A, None) == L.ERR_INVALID and "divisible by 32" in _msg(lib)
    assert q(4, A, L.X_BF16, 256, 0, 256, A, A, None) == L.ERR_INVALID
    assert q(4, A, L.X_BF16, 128, 2, 256, A, A, None) == L.ERR_INVALID and "ldx" in _msg(lib)
    assert q(4, ODD, L.X_BF16, 256, 1, 256, A, A, None) == L.ERR_INVALID
    assert q(4, A, L.X_BF16, 256, 1, 256, ODD, A, None) == L.ERR_INVALID and "aligned" in _msg(lib)
    assert q(4, A, L.X_F32, 1 << 20, 1 << 30, 1 << 20, A, A, None) == L.ERR_UNSUPPORTED
    d = lib.mfq_hip_mx_dequant_quantized
    assert d(6, A, A, 1, 256, 9, A, 256, None) == L.ERR_INVALID and "out_dtype" in _msg(lib)
    assert d(6, A, A, 2, 256, L.X_F32, A, 255, None) == L.ERR_INVALID and "ldo" in _msg(lib)
    assert d(6, None, A, 2, 256, L.X_F32, A, 256, None) == L.ERR_INVALID
    assert lib.mfq_hip_mx_lay_scales(A, 4, 40, A, None) == L.ERR_INVALID and lib.mfq_hip_mx_lay_scales(A, 4, 64, ODD, None) == L.ERR_INVALID


def gemm(lib, **k):
    a = dict(values=A, scales=A, rows=64, cols=256, row0=0, nrows=64, act=4, x=A, xd=L.X_BF16, ldx=256, xs=None, M=2, glu=0, activation=0, y=A, yd=L.X_F32,
             ldy=64, ws=None, nbytes=0)
    a.update(k)
    return lib.mfq_hip_mx_scaled_gemm_rows(*a.values(), None)


@pytest.mark.parametrize("change,status,word", [
    (dict(values=None), "INVALID", "null"), (dict(act=8), "INVALID", "kind 8"), (dict(xd=5), "INVALID", "x_dtype"), (dict(yd=5), "INVALID", "y_dtype"),
    (dict(cols=100), "INVALID", "divisible by 32"), (dict(values=ODD), "INVALID", "16-byte"), (dict(xs=A, x=ODD), "INVALID", "quantised activations"),
    (dict(ldx=128), "INVALID", "ldx"), (dict(ldy=63), "INVALID", "ldy"), (dict(M=0), "INVALID", "M=0"), (dict(row0=1), "INVALID", "rows 1 + 64 of 64"),
    (dict(glu=1), "INVALID", "16-bit"), (dict(glu=1, yd=L.X_BF16, activation=4), "INVALID", "activation=4"),
    (dict(glu=1, yd=L.X_BF16, nrows=63), "INVALID", "gate and up"), (dict(y=ODD), "INVALID", "unaligned y"), (dict(x=ODD), "INVALID", "unaligned x"),
    (dict(rows=1 << 20, nrows=1 << 20, cols=1 << 13, ldx=1 << 13, ldy=1 << 20), "UNSUPPORTED", "weights"),
    (dict(M=20), "WORKSPACE", "workspace"), (dict(M=20, ws=A, nbytes=20 * 128), "WORKSPACE", "workspace"),
    (dict(M=20, ws=ODD, nbytes=1 << 20), "WORKSPACE", "unaligned")])
def test_gemm_checks(lib, change, status, word):
    assert gemm(lib, **change) == getattr(L, "ERR_" + status), _msg(lib)
    assert word in _msg(lib)


def moe(lib, **k):
    a = dict(values=A, scales=A, rows=256, cols=256, out=64, slot=None, E=4, act=6, x=A, xd=L.X_BF16, ldx=256, xs=None, routed=0, ids=A, T=2, R=2, dst=None,
             bounds=None, glu=0, activation=0, y=A, yd=L.X_F32, ldy=64, ws=None, nbytes=0)
    a.update(k)
    return lib.mfq_hip_mx_moe_matmul(*a.values(), None)


@pytest.mark.parametrize("change,status,word", [
    (dict(ids=None), "INVALID", "ids"), (dict(dst=A), "INVALID", "both ids_dst and expert_bounds"), (dict(T=0), "INVALID", "0 tokens"),
    (dict(E=5), "INVALID", "not 5 experts"), (dict(out=60), "INVALID", "not 4 experts"), (dict(act=8), "INVALID", "kind 8"),
    (dict(glu=1, yd=L.X_F16, out=64, activation=9), "INVALID", "activation=9"), (dict(ldy=10), "INVALID", "ldy"), (dict(ldx=255), "INVALID", "ldx"),
    (dict(T=1 << 16, R=1 << 15), "INVALID", "tokens"), (dict(T=40000, R=2), "UNSUPPORTED", "without a route map"),
    (dict(dst=A, bounds=A, cols=8192, ldx=8192), "WORKSPACE", "workspace"), (dict(T=1000, xs=A, dst=A, bounds=A), "WORKSPACE", "workspace"), (dict(dst=A, bounds=A, cols=8192, ldx=8192, ws=ODD, nbytes=1 << 20), "WORKSPACE", "unaligned"),
    (dict(T=1 << 20, R=16, routed=1, dst=A, bounds=A, ws=A, nbytes=1 << 40), "UNSUPPORTED", "rows of activations")])
def test_moe_checks(lib, change, status, word):
    assert moe(lib, **change) == getattr(L, "ERR_" + status), _msg(lib)
    assert word in _msg(lib)


def test_columns_beyond_the_tiles_offsets(lib):
    K = (1 << 24) + 32
    assert gemm(lib, cols=K, ldx=K, rows=2, nrows=2, M=200, ws=A, nbytes=1 << 50) == L.ERR_UNSUPPORTED and f"{K} columns" in _msg(lib)
    assert moe(lib, cols=K, ldx=K, rows=4, out=1, ldy=1) == L.ERR_UNSUPPORTED and f"{K} columns" in _msg(lib)


def test_scales_are_laid_where_they_are():
    """laid_scales launches on the current GPU: a weight that is elsewhere is refused before anything runs."""
    w = MxWeight(F.MxHeader("MXFP4", 4, 64, 256, 0, 64 * 128, 64 * 128, 64 * 8), torch.zeros(64, 128, dtype=torch.uint8), torch.zeros(64, 8, dtype=torch.uint8))
    with pytest.raises(ValueError, match="on the current GPU, got cpu"):
        w.laid_scales()
    with pytest.raises(ValueError, match="on the current GPU, got cpu"):
        mx_scaled_matmul(w, torch.zeros(2, 256))


def test_noted_workspaces_stay_few():
    w = MxWeight(F.MxHeader("MXFP4", 4, 64, 256, 0, 64 * 128, 64 * 128, 64 * 8), torch.zeros(64, 128, dtype=torch.uint8), torch.zeros(64, 8, dtype=torch.uint8))
    assert [w.note_need(m, 2 * m) for m in range(5000)] == [2 * m for m in range(5000)] and 0 < len(w._needs) <= 1024


def test_oracle_quantiser_closed_forms():
    """Grids, the scale rule and ties, written out by hand."""
    assert P.E2M1.tolist() == [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    assert P.E2M3[:9].tolist() == [0, 0.125, 0.25, 0.375, 0.5, 0.625, 0.75, 0.875, 1] and P.E2M3[31] == 7.5 and P.E2M3[24] == 4
    x = np.zeros((1, 32))
    x[0, :8] = [4.0, 0.25, 0.75, 2.5, 3.5, 5.0, -5.5, 7.9]      # exponent 2: scale 1
    codes, scale = P.quantize(x, "MXFP4")
    assert scale[0, 0] == 127 and P.values(codes, scale, "MXFP4")[0, :8].tolist() == [4, 0, 1, 2, 4, 4, -6, 6]
    codes, scale = P.quantize(x, "MXFP6")
    assert scale[0, 0] == 127 and P.values(codes, scale, "MXFP6")[0, :8].tolist() == [4, 0.25, 0.75, 2.5, 3.5, 5, -5.5, 7.5]
    x[0, 3] = np.inf
    codes, scale = P.quantize(x, "MXFP6")
    assert scale[0, 0] == 255 and not codes.any()
    codes, scale = P.quantize(np.full((1, 32), 2.0 ** -140), "MXFP4")
    assert scale[0, 0] == 0 and not codes.any()


def test_oracle_packs_what_it_unpacks():
    rng = np.random.default_rng(1)
    codes = rng.integers(0, 64, (3, 288), dtype=np.uint8)
    packed = P.pack(codes, "MXFP6").reshape(3, 2, 192)
    block = np.concatenate([packed[:, 1, :16], packed[:, 1, 128:136]], 1)      # block 8: columns 256 .. 287
    bits = np.unpackbits(block, axis=1, bitorder="little").reshape(3, 32, 6)
    assert np.array_equal((bits << np.arange(6)).sum(-1), codes[:, 256:])
    codes4 = codes & 15
    assert np.array_equal(P.unpack(P.pack(codes4, "MXFP4"))[:, :288], codes4)
