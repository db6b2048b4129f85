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


@pytest.mark.parametrize("pages", BOTH)
def test_pages_outside_the_cache_of_rows_that_stay(dev, pages):
    """Also where the number of the page's holders does not change."""
    w = Rows(4, 5, pages, 4)
    w.grow([9, 4, 0, 18])
    for bad in (-1, pages, -(1 << 31), (1 << 31) - 1):
        for r, c in ((0, 0), (0, 2), (3, 4)):                 # full pages and last ones
            table, free, state, shares, lens = w.tensors(dev)
            table[r, c] = bad
            refused(dev, table, free, state, shares, lens, [0, 1, 2, 3], 4, 64)
        table, free, state, shares, lens = w.tensors(dev, fill=bad)       # behind the rows' pages there is nothing to refuse
        assert blockedAttention.pagedFork(table, free, state, shares, lens, torch.arange(4, device=dev), 4)[2].tolist() == [len(w.free), 0]


@pytest.mark.parametrize("pages", BOTH)
@pytest.mark.parametrize("first,second", [(3, 4), (3, 12), (12, 3), (0, 19)])
def test_counts_that_are_too_low(dev, pages, first, second):
    """Two rows hold a page of which `shares` knows one: what counts is where the count ends, not how it gets there."""
    i32, i64 = dict(dtype=torch.int32, device=dev), dict(dtype=torch.int64, device=dev)
    n = 20
    table = torch.arange(n, **i32)[:, None].repeat(1, 3)
    table[:, 1:] = -1
    table[second, 0] = table[first, 0]
    lens, shares = torch.full((n,), 4, **i64), torch.zeros(pages, **i32)
    free, state = torch.full((pages,), -7, **i32), torch.zeros(2, **i64)
    others = [r for r in range(n) if r not in (first, second)]
    # one ends and two more go on from the other: 0 - 1 + 2; the pages of the two are free
    origin = torch.arange(n, device=dev)
    origin[first], origin[others[0]], origin[others[9]] = -1, second, second
    for _ in range(10):
        free.fill_(-7)
        got = blockedAttention.pagedFork(table, free, state, shares, lens, origin, 4)
        assert got[2].tolist() == [2, 0]
        assert got[3][first].item() == 1 and got[3].sum().item() == 1
        assert free[:2].tolist() == sorted([others[0], others[9]]) and (free[2:] == -7).all()
        assert got[0][second, 0].item() == got[0][others[9], 0].item() == first
    # both end: -2
    origin = torch.arange(n, device=dev)
    origin[first] = origin[second] = -1
    for _ in range(10):
        refused(dev, table, free, state, shares, lens, origin.tolist(), 4, 64)
