"""Refusals beside those of test_mx8_errors.py: sizes whose launches would have 2^32 threads or more, which no device takes.  All before anything is
launched, so they need no GPU."""
import pytest

from test_mx8_errors import P, gemm, lib, logprobs, moe, refused      # noqa: F401 (lib is a fixture)
from tyloquant_amd import _lib as L

ROOM = 1 << 60      # bytes of a workspace


@pytest.mark.parametrize("kw", [dict(M=1 << 24), dict(M=(1 << 31) - 1, top=0), dict(M=1 << 24, V=1, ldl=1, top=1, dtype=0)])
def test_rows_of_logits(lib, kw):
    refused(lib, logprobs(lib, **kw), L.ERR_UNSUPPORTED, "rows")


def test_values_that_a_product_quantises(lib):
    refused(lib, gemm(lib, cols=512, ldx=512, M=(1 << 29) - 1, bytes=ROOM), L.ERR_UNSUPPORTED, "values")
    refused(lib, lib.mfq_hip_mx8_quantize_rows(P, 0, 512, (1 << 29) - 1, 512, P, P, None), L.ERR_UNSUPPORTED, "values")


@pytest.mark.parametrize("kw", [
    dict(rows=65536, nrows=65536, cols=128, ldy=65536, M=1 << 27, x_scales=P),                      # quantised rows
    dict(rows=65536, nrows=65536, cols=128, ldy=65536, ldx=128, M=1 << 28, bytes=ROOM),             # rows that would be quantised first
    dict(rows=65536, nrows=65536, cols=128, ldy=65536, M=1 << 27, x_scales=P, glu=1),
])
def test_tiles_of_a_product(lib, kw):
    refused(lib, gemm(lib, **kw), L.ERR_UNSUPPORTED, "tiles")


@pytest.mark.parametrize("kw", [
    dict(dst=None, bounds=None, cols=128, ldx=128, T=1 << 24, R=8),                                  # a block or more a pair
    dict(cols=128, ldx=128, rows=4 << 23, out=1 << 23, ldy=1 << 23, T=1 << 20, R=8, bytes=ROOM),     # tiles of a route map
])
def test_tiles_of_experts(lib, kw):
    refused(lib, moe(lib, **kw), L.ERR_UNSUPPORTED, "tiles")


def test_no_kernel_for_pairs_of_long_rows(lib):
    """the host's limit is the one that a call without a route map is held to"""
    from tyloquant_amd import runtime_mx8 as R8
    most = R8.MAX_PAIR_COLUMNS
    assert [lib.mfq_hip_mx8_moe_plan(K, 8, 4, 0) for K in (128, most, most + 128)] == [0, 0, -1]
    assert lib.mfq_hip_mx8_moe_plan(most + 128, 8, 4, 1) > 0
    refused(lib, moe(lib, dst=None, bounds=None, cols=most + 128, ldx=most + 128), L.ERR_UNSUPPORTED, "without a route map")
