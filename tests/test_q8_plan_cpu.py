"""The launch rules of the 8-bit products on the CPU: sizes that no test can hold."""
import pytest

from tests import q8_plan
from tests.q8_plan import FITS, WIDE, plan


@pytest.mark.parametrize('out_bytes', [2, 4])
@pytest.mark.parametrize('K', [16, 128, 144, 1024])
def test_rows_of_a_result_fit_the_stores(K, out_bytes):
    """A lane's place behind the first of 32 rows and 64 columns is (4 n_cols + 62) numbers, kept in 32 bits: wider results are refused,
    for any number of rows."""
    top = q8_plan.library().max_cols()
    assert 4 * top + 62 < 2 ** 31 and (4 * top + 62) * 4 < 2 ** 32
    for M in (1, 31, 64, 300):
        assert plan(M, top, K, out_bytes).refusal != WIDE
        for n in (top + 1, 2 ** 28, 2 ** 29, 2 ** 31 - 1):
            assert plan(M, n, K, out_bytes).refusal == WIDE
            assert plan(M, n, K, out_bytes, n_seg=5, ragged=True).refusal == WIDE
    assert plan(64, top, K, out_bytes).refusal == FITS
