"""pagedFork where `shares` and the table's pages do not fit: refused as a whole, by one workgroup and by three launches alike."""
import pytest
import torch

import blockedAttention
from test_gpu_paged_fork import Rows, refused

pytestmark = pytest.mark.gpu

BOTH = [40, 20000, (1 << 20) + 70]                            # pages: one workgroup; three launches with chunks of either size


@pytest.mark.parametrize("pages", BOTH)
@pytest.mark.parametrize("value", [-1, -2, -(1 << 31)])
@pytest.mark.parametrize("origin", [[0, 1, 2, 3], [-1, 1, 2, -1], [0, 0, 0, 3]])
def test_counts_below_zero(dev, pages, value, origin):
    """On a page of a row that stays, of one that ends, and on those that nobody holds, at both ends and in the middle."""
    w = Rows(4, 5, pages, 4)
    w.grow([9, 4, 0, 18])
    held = {p for row in w.rows for p in row}
    loose = [p for p in (0, pages // 2, pages - 1) if p not in held]
    for where in (w.rows[1][0], w.rows[3][0], *loose):
        table, free, state, shares, lens = w.tensors(dev)
        shares[where] = value
        refused(dev, table, free, state, shares, lens, origin, 4, 64)
