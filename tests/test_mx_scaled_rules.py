"""Rules of the products of microscaled operands on the host: sizes at their ends, and which kernel a call takes (nothing is launched)."""
import pytest

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
