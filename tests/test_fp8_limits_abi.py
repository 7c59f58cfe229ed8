"""Limits of the 8-bit quantiser's launches, on the host: every check comes before the first use of the device."""
import pytest

from tests.test_fp8_abi import A, both, quantize


@pytest.mark.parametrize("K", [(1 << 28) - 63, 1 << 28, 1 << 29])
def test_column_sums_of_too_many_columns_are_refused(K):
    """A workgroup of 1024 threads sums 64 columns: 2^28 columns are 2^32 threads."""
    sums = dict(colsum=A, ws=A, nws=4 * K)
    assert quantize(R=1, K=K, ldx=K, transpose=1, ldq=128, **sums) == -1
    assert both(R=1, K=K, ldx=K, ldq=(K + 127) // 128 * 128, lds=1 << 24, **sums) == -1
