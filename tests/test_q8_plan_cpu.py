"""The launch rules of the 8-bit products on the CPU: sizes that no test can hold."""
import ctypes
import random

import pytest

from tests import q8_plan, q8_reach
from tests.q8_plan import FEW, FITS, LONG, SHORT, WIDE, plan


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


@pytest.mark.parametrize('out_bytes', [2, 4])
@pytest.mark.parametrize('K,widest', [(16, 65535 * 128), (128, 65535 * 128), (256, 65535 * 128), (272, 65535 * 32), (4096, 65535 * 32)])
def test_few_rows_of_any_width(K, widest, out_bytes):
    """The kernel for few rows has its column tiles in the grid's second dimension, 65535 of them; wider results go to the others."""
    for M in (1, 2, 33, 63):
        p = plan(M, widest, K, out_bytes)
        assert p.refusal == FITS and p.kernel == FEW and p.grid_y == 65535
        for n in (widest + 1, 10 * widest, q8_plan.library().max_cols()):
            p = plan(M, min(n, q8_plan.library().max_cols()), K, out_bytes)
            assert p.refusal == FITS and p.kernel == (SHORT if K <= 128 else LONG) and p.grid_y == 1


@pytest.mark.parametrize('out_bytes', [2, 4])
def test_what_fits_the_memory_is_launched(out_bytes):
    """Products of one segment of up to 2^30 - 1024 rows whose operands and result fit 288 GB, and launches within the grid's limits that cover every result."""
    rng = random.Random(out_bytes)
    seen = set()
    for _ in range(20000):
        M, n, K = (int(2 ** rng.uniform(0, top)) for top in (30, 27, 16))
        M, K = min(M, 2 ** 30 - 1024), max(16, K // 16 * 16)
        if (M + n) * K + M * n * out_bytes > 288e9:
            continue
        p = plan(M, n, K, out_bytes)
        assert p.refusal == FITS, (M, n, K)
        seen.add(p.kernel)
        if p.kernel == FEW:
            rows, cols, threads = 32 if p.split else 128 // p.across, 32 if p.split else 32 * p.across, 256
            assert p.grid_x == p.tiles and p.grid_y == p.cuts <= 65535
        else:
            rows, cols, threads = (32 * p.rt, 64 * p.wc, 512) if p.kernel == SHORT else (128, 128, 256)
            assert p.grid_x >= p.tiles * p.cuts and p.grid_x % 8 == 0 and p.grid_y == 1
        assert p.tiles * rows >= M and p.cuts * cols >= n and p.grid_x * threads < 2 ** 32 and p.tiles * p.cuts < 2 ** 31
    assert seen == {FEW, SHORT, LONG}


def test_rows_are_counted_in_an_int():
    """The furthest row that a kernel names is 1023 past the last (score: 8 waves of 4 x 32 pixels from the tile's first on)."""
    lib = q8_plan.library()
    top = 2 ** 31 - 1024
    assert 7 * 4 * 32 + 3 * 32 + 31 == 1023 and top - 1 + 1023 < 2 ** 31
    for n, fits in ((top, 1), (top + 1, 0), (2 ** 31 - 1, 0), (2 ** 31, 0), (2 ** 32 + 1, 0), (2 ** 40, 0)):
        assert lib.rows_fit(ctypes.c_int64(n)) == fits


def test_sizes_of_the_gpu_tests_reach_each_kernel():
    for sizes, kernel in ((q8_reach.FEW, FEW), (q8_reach.SHORT, SHORT), (q8_reach.LONG, LONG)):
        for m, n, k in sizes:
            for out_bytes in (2, 4):
                assert plan(m, n, k, out_bytes).kernel == kernel, (m, n, k)
    assert {plan(*s).split for s in q8_reach.FEW} == {0, 1} and {plan(*s).across for s in q8_reach.FEW} == {1, 4}
    assert any(k % 128 for _, _, k in q8_reach.SHORT) and any(k % 128 for _, _, k in q8_reach.LONG)
    # the score: 256-pixel workgroups from half the compute units on
    for sizes, lds in ((q8_reach.SCORES_FEW, False), (q8_reach.SCORES_LDS, True)):
        for n, h, w, d in sizes:
            assert (2 * n * -(-h * w // 256) >= 256) == lds
