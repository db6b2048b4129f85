"""pagedFork against the same rules in Python: lists of pages, counts of who holds them, and a stack."""
import pytest
import torch

import blockedAttention

pytestmark = pytest.mark.gpu


class Rows:
    """A table whose pages may be shared, on the host."""

    def __init__(self, rows, width, pages, page, seed=0):
        self.g = torch.Generator().manual_seed(seed)
        self.page, self.width, self.pages = page, width, pages
        self.lens, self.rows, self.shares = [0] * rows, [[] for _ in range(rows)], [0] * pages
        self.free = torch.randperm(pages, generator=self.g).tolist()

    def grow(self, new):
        """As pagedResize does for rows that get longer."""
        for r, n in enumerate(new):
            assert n >= self.lens[r]
            while len(self.rows[r]) < -(-n // self.page):
                self.rows[r].append(self.free.pop())
            self.lens[r] = n

    def fork(self, origin):
        page, lens, rows = self.page, self.lens, self.rows
        kept = {o for r, o in enumerate(origin) if o == r}
        new, copies, source, target = [], [], [-1] * len(rows), [-1] * len(rows)
        for r, o in enumerate(origin):
            row = list(rows[o]) if o >= 0 else []
            if row and lens[o] % page and o != r:
                if o in kept:
                    copies.append(r)
                    row[-1] = None
                kept.add(o)
            new.append(row)
        holders = [0] * self.pages
        for p in (p for row in new for p in row if p is not None):
            holders[p] += 1
        held = {p for row in rows for p in row}
        stack = self.free + [p for p in sorted(held) if holders[p] == 0]
        if len(copies) > len(stack):
            return False, source, target
        for r in copies:
            source[r], target[r] = rows[origin[r]][-1], stack.pop()
            new[r][-1] = target[r]
            holders[target[r]] = 1
        for p in held | set(target) - {-1}:
            self.shares[p] = max(0, holders[p] - 1)
        self.free, self.rows, self.lens = stack, new, [lens[o] if o >= 0 else 0 for o in origin]
        return True, source, target

    def tensors(self, dev, fill=-1):
        i32 = dict(dtype=torch.int32, device=dev)
        table = torch.full((len(self.rows), self.width), fill, **i32)
        for r, row in enumerate(self.rows):
            table[r, :len(row)] = torch.tensor(row, **i32)
        free = torch.full((self.pages,), -7, **i32)
        free[:len(self.free)] = torch.tensor(self.free, **i32)
        return table, free, torch.tensor([len(self.free), 0], device=dev), torch.tensor(self.shares, **i32), torch.tensor(self.lens, device=dev)

    def check(self, got, free, stack_before, source, target):
        table, lens, state, shares, src, dst = got
        assert state.tolist() == [len(self.free), 0]
        assert lens.tolist() == self.lens and src.tolist() == source and dst.tolist() == target
        assert shares.tolist() == self.shares
        assert free[:len(self.free)].tolist() == self.free
        assert torch.equal(free[max(len(self.free), stack_before):], torch.full_like(free[max(len(self.free), stack_before):], -7))
        want = torch.full(table.shape, -1, dtype=torch.int32)
        for r, row in enumerate(self.rows):
            want[r, :len(row)] = torch.tensor(row, dtype=torch.int32)
        assert torch.equal(table.cpu(), want)


def origins(kind, n, g):
    if kind == "stay":
        return list(range(n))
    if kind == "end":
        return [-1] * n
    if kind == "one":                                         # all go on from one row, which itself becomes another's
        return [n // 2] * n
    if kind == "swap":
        return list(range(n))[::-1]
    return torch.randint(-1, n, (n,), generator=g).tolist()


@pytest.mark.parametrize("rows,width,pages,page,longest", [(1, 4, 9, 16, 60), (5, 6, 60, 1, 6), (32, 40, 2000, 16, 500), (300, 9, 9000, 7, 60), (70, 300, 60000, 4, 1100),
                                                           (1500, 3, 20000, 5, 14)])
def test_steps(dev, rows, width, pages, page, longest):
    """Several steps one after the other: rows fork, grow by some tokens, fork again."""
    w = Rows(rows, width, pages, page)
    g = w.g
    w.grow(torch.randint(0, longest + 1, (rows,), generator=g).tolist())
    for kind in ("any", "stay", "any", "one", "any", "swap", "any", "end"):
        table, free, state, shares, lens = w.tensors(dev, fill=12345)
        before = [t.clone() for t in (table, state, shares, lens)]
        stack = len(w.free)
        origin = origins(kind, rows, g)
        fine, source, target = w.fork(origin)
        assert fine
        o = torch.tensor(origin, device=dev)
        got = blockedAttention.pagedFork(table, free, state, shares, lens, o, page)
        w.check(got, free, stack, source, target)
        again = blockedAttention.pagedFork(table, free, state, shares, lens, o, page)
        assert all(torch.equal(a, b) for a, b in zip(got, again))
        assert all(torch.equal(a, b) for a, b in zip(before, (table, state, shares, lens)))
        if kind in ("any", "swap"):
            room = sum(1 for _ in w.free)
            new, used = [], 0
            for n, row in zip(w.lens, w.rows):
                n2 = min(n + int(torch.randint(0, 9, (1,), generator=g)), width * page)
                need = -(-n2 // page) - len(row)
                if used + need > room - rows:
                    n2, need = n, 0
                used += need
                new.append(n2)
            w.grow(new)


def test_fresh_pages_come_from_the_freed_ones_too(dev):
    """An empty stack: rows that end give their pages to the copies, the largest number first."""
    w = Rows(6, 5, 30, 4)
    w.free = list(range(30))[::-1]
    w.grow([20, 20, 20, 20, 18, 3])
    w.free = w.free[:0]
    w.pages = 30
    table, free, state, shares, lens = w.tensors(dev)
    origin = [-1, 4, 4, -1, 4, 5]
    fine, source, target = w.fork(origin)
    assert fine and sorted(target)[-2:] == [18, 19]
    w.check(blockedAttention.pagedFork(table, free, state, shares, lens, torch.tensor(origin, device=dev), 4), free, 0, source, target)


def test_freed_pages_of_many_chunks(dev):
    """Fresh pages are looked up among freed ones that lie far apart."""
    rows, page = 600, 3
    w = Rows(rows, 200, 700000, page)
    w.grow([550 + r % 7 for r in range(rows)])
    w.free = w.free[:0]
    table, free, state, shares, lens = w.tensors(dev)
    origin = [-1 if r % 5 == 0 else (r // 5 * 5 + 1) for r in range(rows)]
    fine, source, target = w.fork(origin)
    assert fine
    w.check(blockedAttention.pagedFork(table, free, state, shares, lens, torch.tensor(origin, device=dev), page), free, 0, source, target)


def refused(dev, table, free, state, shares, lens, origin, page, verdict):
    before = [t.clone() for t in (table, free, state, shares, lens)]
    got = blockedAttention.pagedFork(table, free, state, shares, lens, torch.tensor(origin, device=dev), page)
    assert got[2].tolist() == [before[2][0].item(), verdict]
    assert torch.equal(got[0], before[0]) and torch.equal(got[1], before[4]) and torch.equal(got[3], before[3])
    assert (got[4] == -1).all() and (got[5] == -1).all()
    assert all(torch.equal(a, b) for a, b in zip(before, (table, free, state, shares, lens)))


@pytest.mark.parametrize("pages", [40, 20000])                # one workgroup does all of it, or three launches
def test_refusals_change_nothing(dev, pages):
    w = Rows(4, 5, pages, 4)
    w.grow([9, 4, 0, 18])
    w.free = w.free[:2]
    fresh = lambda **change: [change.get(n, t) for n, t in zip(("table", "free", "state", "shares", "lens"), w.tensors(dev))]  # noqa: E731
    table, free, state, shares, lens = w.tensors(dev)
    refused(dev, *fresh(free=free[:2].clone()), [0, 0, 0, 3], 4, 16)      # freed pages beyond the stack
    refused(dev, *fresh(), [0, 3, 4, 3], 4, 32)
    refused(dev, *fresh(), [0, 3, -2, 3], 4, 32)
    refused(dev, *fresh(), [0, 3, 1 << 40, 3], 4, 32)
    refused(dev, *fresh(lens=torch.tensor([9, 4, -1, 18], device=dev)), [0, 1, 2, 3], 4, 4)
    refused(dev, *fresh(lens=torch.tensor([9, 4, 21, 18], device=dev)), [0, 1, 2, 3], 4, 4)
    refused(dev, *fresh(lens=torch.tensor([9, 4, 21, 18], device=dev)), [0, 1, 2, 9], 4, 36)
    refused(dev, *fresh(state=torch.tensor([-1, 0], device=dev)), [0, 1, 2, 3], 4, 16)
    refused(dev, *fresh(state=torch.tensor([pages + 1, 0], device=dev)), [0, 1, 2, 3], 4, 16)
    refused(dev, *fresh(state=torch.tensor([2, 8], device=dev)), [0, 1, 2, 3], 4, 8)
    for page in (-1, pages, -(1 << 31), (1 << 31) - 1):
        bad = table.clone()
        bad[3, 1] = page
        refused(dev, *fresh(table=bad), [0, 1, 2, -1], 4, 64)
    bad = table.clone()
    bad[3, 1] = bad[3, 0]                                     # the same page twice, held once
    refused(dev, *fresh(table=bad), [0, 1, 2, -1], 4, 64)


@pytest.mark.parametrize("pages", [40, 20000])
def test_too_few_pages(dev, pages):
    w = Rows(5, 5, pages, 4)
    w.grow([9, 4, 0, 0, 0])
    for n, verdict in ((3, 0), (2, 1), (0, 1)):
        table, free, state, shares, lens = w.tensors(dev)
        state[0] = n
        if verdict:
            refused(dev, table, free, state, shares, lens, [0, 1, 0, 0, 0], 4, 1)
        else:
            got = blockedAttention.pagedFork(table, free, state, shares, lens, torch.tensor([0, 1, 0, 0, 0], device=dev), 4)
            assert got[2].tolist() == [0, 0]
    refused(dev, table, free, torch.tensor([2, 0], device=dev), shares, lens, [0, 0, 0, 0, 0], 4, 1)       # four copies; row 1 gives one page back
    got = blockedAttention.pagedFork(table, free, torch.tensor([3, 0], device=dev), shares, lens, torch.tensor([0, 0, 0, 0, 0], device=dev), 4)
    assert got[2].tolist() == [0, 0]


def test_empty_tables(dev):
    i64, i32 = dict(dtype=torch.int64, device=dev), dict(dtype=torch.int32, device=dev)
    got = blockedAttention.pagedFork(torch.zeros((0, 4), **i32), torch.zeros(3, **i32), torch.tensor([2, 0], **i64), torch.zeros(5, **i32), torch.zeros(0, **i64),
                                     torch.zeros(0, **i64), 16)
    assert got[0].shape == (0, 4) and got[2].tolist() == [2, 0] and got[3].tolist() == [0] * 5
    got = blockedAttention.pagedFork(torch.zeros((3, 0), **i32), torch.zeros(0, **i32), torch.tensor([0, 0], **i64), torch.zeros(0, **i32), torch.zeros(3, **i64),
                                     torch.tensor([2, -1, 0], **i64), 16)
    assert got[1].tolist() == [0, 0, 0] and got[2].tolist() == [0, 0]


@pytest.mark.parametrize("pages", [2000, 20000])
def test_in_a_graph_and_on_another_stream(dev, pages):
    w = Rows(40, 20, pages, 8, seed=4)
    w.grow(torch.randint(0, 150, (40,), generator=w.g).tolist())
    table, free, state, shares, lens = w.tensors(dev)
    origin = torch.arange(40, device=dev)
    call = lambda: blockedAttention.pagedFork(table, free, state, shares, lens, origin, 8)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    side = torch.cuda.Stream()
    first = (w.lens, w.rows, list(w.shares), list(w.free))
    for step in range(5):
        w.lens, w.rows, w.shares, w.free = first[0], first[1], list(first[2]), list(first[3])
        o = origins("any", 40, w.g)
        origin.copy_(torch.tensor(o))
        free.copy_(w.tensors(dev)[1])
        fine, source, target = w.fork(o)
        assert fine
        graph.replay()
        torch.cuda.synchronize()
        w.check(out, free, len(first[3]), source, target)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = call()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, again))


def test_most_rows(dev):
    w = Rows(8192, 2, 60000, 4, seed=9)
    w.grow(torch.randint(0, 9, (8192,), generator=w.g).tolist())
    table, free, state, shares, lens = w.tensors(dev)
    stack = len(w.free)
    o = origins("any", 8192, w.g)
    fine, source, target = w.fork(o)
    assert fine
    w.check(blockedAttention.pagedFork(table, free, state, shares, lens, torch.tensor(o, device=dev), 4), free, stack, source, target)
    i64, i32 = dict(dtype=torch.int64, device=dev), dict(dtype=torch.int32, device=dev)
    with pytest.raises(RuntimeError, match="up to 8192 rows"):
        blockedAttention.pagedFork(torch.zeros((8193, 2), **i32), free, state, shares, torch.zeros(8193, **i64), torch.zeros(8193, **i64), 4)


def test_more_than_a_million_pages(dev):
    """Pages at both ends of a large cache, with chunks of the other size."""
    w = Rows(50, 40, (1 << 20) + 70, 4, seed=11)
    w.grow(torch.randint(0, 160, (50,), generator=w.g).tolist())
    for kind in ("any", "one", "end"):
        table, free, state, shares, lens = w.tensors(dev)
        stack, o = len(w.free), origins(kind, 50, w.g)
        fine, source, target = w.fork(o)
        assert fine
        w.check(blockedAttention.pagedFork(table, free, state, shares, lens, torch.tensor(o, device=dev), 4), free, stack, source, target)
