"""The paged attention at the ends of its numbers: E4M3 rows whose powers of two lie
far apart (the plain forms are those of test_gpu_paged.py).
"""

import numpy as np
import pytest

from test_gpu_paged import Case, attend, check, ctx  # noqa: F401 (ctx: the fixture)

pytestmark = pytest.mark.gpu


def test_a_bad_page_beside_rows_of_far_powers(ctx):  # noqa: F811
    # In a tile of keys whose value rows' powers lie far apart a page is none: rows that
    # see none of its keys are as they were, whatever the pool's first page holds.
    case = Case("E4M3", [70], [140], 384, 1, 64, 16, seed=227, noise=0.0, spare_pages=3)
    spare = int(np.setdiff1d(np.arange(case.pages), case.table)[-1])
    for rows in (case.key_rows, case.value_rows):
        rows[[0, spare]] = rows[[spare, 0]]
    case.table[case.table == 0] = spare
    case.value_rows *= np.float32(2.0 ** 12)       # the first row's power is large
    case.value_rows[case.table[0, 4], :, 1] = 0     # position 65
    case.quantise()
    case.value_exponents[0] = case.key_exponents[0] = 0
    clean = check(ctx, case)
    case.table[0, 7] = -1                           # positions 112 on
    got = attend(ctx, case)
    assert np.isnan(got[112 - 70:]).all()
    assert np.array_equal(got[:112 - 70], clean[:112 - 70])
