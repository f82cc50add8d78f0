"""The operators of a batched step over a paged 8-bit cache at the ends of what their header allows, against the 64-bit
forms of serving_ref.py, within test_gpu_serving's bound unless one is derived here."""
import numpy as np
import pytest

import serving_ref as R
from test_gpu_serving import check_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("q", [1, 6, 90])
def test_pages_that_are_not_there_beside_codes_that_are_no_numbers(q, half):
    """Page 0 belongs to no sequence and holds NaN codes, as memory that nothing was stored to may."""
    rng = np.random.default_rng(14)

    def bad(codes, scale, table, q):
        unused = np.setdiff1d(np.arange(1, codes.shape[1]), table)
        table[table == 0] = unused[0]
        codes[:, 0], scale[:, 0] = 0x7F, np.nan
        table[0, 2], table[0, 5], table[1, 0], table[2, :] = -1, 2 ** 31 - 1, codes.shape[1], -2 ** 31

    got = check_attention(rng, 8, 2, 128, 16, [200, 100, 95], [q, q, q], R.E4M3, half, change=bad)
    assert (got[2 * q:3 * q] == 0).all() and np.isfinite(got[:3 * q]).all()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("cache", [R.INT8, R.E4M3])
def test_rows_that_are_not_finite_and_see_no_page(cache, half):
    """Zeros, whatever q holds."""
    rng = np.random.default_rng(15)

    def bad(codes, scale, table, q):
        table[0, :] = -1
        q[3], q[40, :, 5], q[89, 2] = np.nan, np.inf, -np.inf

    got = check_attention(rng, 8, 2, 64, 16, [95, 70], [90, 30], cache, half, change=bad)
    assert (got[:90] == 0).all()
