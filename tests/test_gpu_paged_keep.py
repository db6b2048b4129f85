"""pagedKeep and pagedCopy: what they move arrives bit for bit, and nothing else changes."""
import pytest
import torch

import blockedAttention
from blockedattention_amd import capi

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn
BITS = {torch.float16: torch.int16, torch.bfloat16: torch.int16, FP8: torch.uint8}


def make_cache(dev, dtype, pages, heads, page, dim, order="heads", gap=0, seed=0):
    """Two caches of random bits (NaN among them), rows `gap` elements apart."""
    g = torch.Generator().manual_seed(seed)
    shape = (pages, heads, page, dim + gap) if order == "heads" else (pages, page, heads, dim + gap)
    got = []
    for _ in range(2):
        t = torch.randint(0, 256, (*shape[:-1], shape[-1] * (1 if dtype == FP8 else 2)), generator=g, dtype=torch.uint8).to(dev).view(dtype)
        got.append((t if order == "heads" else t.transpose(1, 2))[..., :dim])
    return got


def bits(t):
    return t.view(torch.uint8) if t.dtype == FP8 else t.view(torch.int16)


def kept(path, base, room):
    """The entries of a path that count."""
    n = 0
    for i, node in enumerate(path):
        if base < 0 or node < i or node <= (path[i - 1] if i else -1) or base + node >= room:
            break
        n += 1
    return n


def expect_keep(cache, table, base, paths, page):
    out = [bits(c).clone() for c in cache]
    lens = []
    for r, path in enumerate(paths):
        n = kept(path, base[r], table.shape[1] * page)
        lens.append(base[r] + n)
        for i in range(n):
            s, d = base[r] + path[i], base[r] + i
            ps, pd = int(table[r, s // page]), int(table[r, d // page])
            if all(0 <= p < len(cache[0]) for p in (ps, pd)):
                for o, c in zip(out, cache):
                    o[pd, :, d % page] = bits(c)[ps, :, s % page]
    return out, lens


@pytest.mark.parametrize("dtype,heads,dim,page,order,gap", [
    (torch.float16, 8, 128, 16, "heads", 0), (torch.bfloat16, 3, 80, 24, "tokens", 0), (FP8, 5, 100, 24, "tokens", 0), (FP8, 2, 3, 1, "heads", 0),
    (torch.float16, 1, 1, 5, "heads", 0), (torch.bfloat16, 4, 37, 7, "heads", 3), (FP8, 33, 64, 16, "heads", 16), (torch.float16, 2, 256, 64, "tokens", 1),
    (FP8, 1, 255, 3, "tokens", 2), (torch.bfloat16, 17, 8, 16, "heads", 0)])
def test_keep(dev, dtype, heads, dim, page, order, gap):
    g = torch.Generator().manual_seed(dim)
    base = [0, 1, page - 1, page, 3 * page + 2, 70, 5]
    nodes = [30, 1, 5, 64, 300, 12, 9]
    depth = 290
    paths = []
    for n in nodes:
        count = int(torch.randint(0, n + 1, (1,), generator=g))
        path = sorted(torch.randperm(n, generator=g)[:count].tolist())
        paths.append(path + [-1] * (depth - len(path)))
    paths[4] = list(range(300))[10:] + []                    # all moved by ten: every source but ten is a target too
    paths[6] = [0, 1, 2, 3] + [-1] * (depth - 4)             # all in place already
    need = [-(-(b + n) // page) for b, n in zip(base, nodes)]
    cache = make_cache(dev, dtype, sum(need) + 2, heads, page, dim, order, gap)
    table = torch.full((len(base), max(need)), -1, dtype=torch.int32)
    order_of, at = torch.randperm(sum(need), generator=g).int(), 0
    for r, n in enumerate(need):
        table[r, :n] = order_of[at:at + n]
        at += n
    want, lens = expect_keep([c.cpu() for c in cache], table, base, paths, page)
    got = blockedAttention.pagedKeep(*cache, table.to(dev), torch.tensor(base, device=dev), torch.tensor(paths, device=dev))
    assert got.tolist() == lens
    for c, w in zip(cache, want):
        assert torch.equal(bits(c).cpu(), w)


@pytest.mark.parametrize("path", [[-1, 5, 6], [3, 3, 4], [3, 2, 7], [0, 0], [2, 4, 1 << 40], [2, 5, 4], [1, 2, 9, 39], [1, 2, 9, 40], [-5], [0, -(1 << 62)], []])
def test_paths_end_where_they_do_not_increase_or_leave_the_row(dev, path):
    page = 10
    cache = make_cache(dev, torch.float16, 9, 2, page, 16)
    table = torch.tensor([[3, 1, 7, 0]], dtype=torch.int32)
    for base in (0, 1, 25, 39, 40, 41, -1, -(1 << 62), 1 << 40):
        want, lens = expect_keep([c.cpu() for c in cache], table, [base], [path], page)
        got = blockedAttention.pagedKeep(*cache, table.to(dev), torch.tensor([base], device=dev), torch.tensor([path], device=dev, dtype=torch.int64).reshape(1, -1))
        assert got.tolist() == lens
        for c, w in zip(cache, want):
            assert torch.equal(bits(c).cpu(), w)


def test_page_numbers_outside_the_cache_are_not_touched(dev):
    cache = make_cache(dev, torch.bfloat16, 4, 2, 4, 16)
    table = torch.tensor([[0, -1, 2], [1, 3, 4], [-(1 << 31), (1 << 31) - 1, 2]], dtype=torch.int32)
    paths = [[1, 4, 8, 9], [2, 4, 9, 10], [5, 8, 9, 10]]
    want, lens = expect_keep([c.cpu() for c in cache], table, [0, 1, 1], paths, 4)
    got = blockedAttention.pagedKeep(*cache, table.to(dev), torch.tensor([0, 1, 1], device=dev), torch.tensor(paths, device=dev))
    assert got.tolist() == lens
    for c, w in zip(cache, want):
        assert torch.equal(bits(c).cpu(), w)


def test_keep_without_requests_or_pages(dev):
    empty = torch.zeros((0, 2, 4, 8), dtype=torch.float16, device=dev)
    none = torch.zeros(0, dtype=torch.int64, device=dev)
    cache = make_cache(dev, torch.float16, 3, 2, 4, 8)
    assert blockedAttention.pagedKeep(*cache, torch.zeros((0, 3), dtype=torch.int32, device=dev), none, none.view(0, 5)).shape == (0,)
    row = torch.zeros((1, 3), dtype=torch.int32, device=dev)
    assert blockedAttention.pagedKeep(empty, empty, row, none.new_tensor([4]), none.new_tensor([[1, 2]])).tolist() == [6]
    assert blockedAttention.pagedKeep(*cache, row[:, :0], none.new_tensor([4]), none.new_tensor([[1, 2]])).tolist() == [4]


def test_keep_writes_no_byte_beside_its_rows(dev):
    """The gaps between rows of a strided cache, by a view of all of it."""
    for dtype in (torch.float16, FP8):
        whole = make_cache(dev, dtype, 6, 3, 8, 61)
        before = [bits(c).clone() for c in whole]
        cache = [c[:, :2, :, 5:42] for c in whole]
        table = torch.tensor([[2, 4]], dtype=torch.int32)
        want, lens = expect_keep([c.cpu() for c in cache], table, [3], [[1, 4, 5, 9]], 8)
        assert blockedAttention.pagedKeep(*cache, table.to(dev), torch.tensor([3], device=dev), torch.tensor([[1, 4, 5, 9]], device=dev)).tolist() == lens
        for c, w, b in zip(whole, want, before):
            b[:, :2, :, 5:42] = w.to(dev)
            assert torch.equal(bits(c), b)


@pytest.mark.parametrize("dtype,heads,dim,page,order,gap", [
    (torch.float16, 8, 128, 16, "heads", 0), (torch.bfloat16, 8, 128, 32, "tokens", 0), (FP8, 5, 100, 24, "tokens", 0), (FP8, 2, 3, 1, "heads", 0),
    (torch.float16, 1, 1, 1, "heads", 0), (torch.bfloat16, 4, 37, 7, "heads", 3), (FP8, 1, 255, 300, "heads", 0), (torch.float16, 3, 40, 24, "tokens", 9),
    (torch.bfloat16, 1, 72, 8, "heads", 8)])
@pytest.mark.parametrize("copies", [1, 40])
def test_copy(dev, dtype, heads, dim, page, order, gap, copies):
    g = torch.Generator().manual_seed(dim)
    pages = 2 * copies + 3
    cache = make_cache(dev, dtype, pages, heads, page, dim, order, gap)
    mixed = torch.randperm(pages, generator=g).int()
    source, target = mixed[:copies].clone(), mixed[copies:2 * copies].clone()
    if copies > 5:
        source[3] = target[3] = -1
        source[5], target[7], target[9], source[11] = pages, -1, -(1 << 31), (1 << 31) - 1
    want = [bits(c).cpu().clone() for c in cache]
    for s, t in zip(source.tolist(), target.tolist()):
        if 0 <= s < pages and 0 <= t < pages:
            for w in want:
                w[t] = w[s]
    assert blockedAttention.pagedCopy(*cache, source.to(dev), target.to(dev)) is None
    for c, w in zip(cache, want):
        assert torch.equal(bits(c).cpu(), w)


def test_copy_writes_no_byte_beside_its_pages(dev):
    for dtype in (torch.float16, FP8):
        for heads, rows in ((slice(0, 2), slice(0, 8)), (slice(0, 3), slice(1, 6)), (slice(1, 2), slice(2, 3))):
            whole = make_cache(dev, dtype, 6, 3, 8, 61)
            before = [bits(c).clone() for c in whole]
            cache = [c[:, heads, rows, 5:42] for c in whole]
            blockedAttention.pagedCopy(*cache, torch.tensor([1, 4], device=dev, dtype=torch.int32), torch.tensor([0, 3], device=dev, dtype=torch.int32))
            for c, b in zip(whole, before):
                b[[0, 3], heads, rows, 5:42] = b[[1, 4], heads, rows, 5:42]
                assert torch.equal(bits(c), b)


def test_copy_of_nothing(dev):
    cache = make_cache(dev, torch.float16, 3, 2, 4, 8)
    before = bits(cache[0]).clone()
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    blockedAttention.pagedCopy(*cache, none, none)
    blockedAttention.pagedCopy(cache[0][:0], cache[1][:0], none.new_tensor([0]), none.new_tensor([1]))
    assert torch.equal(bits(cache[0]), before)


def test_offsets_past_32_bits(dev):
    """Pages whose byte offsets pass 2^32."""
    pages, heads, page, dim = 4200, 8, 256, 256
    cache = [torch.zeros((pages, heads, page, dim), dtype=torch.float16, device=dev) for _ in range(2)]
    for i, c in enumerate(cache):
        c[4199] = 3 + i
        c[4198, :, 200] = 7 + i
    blockedAttention.pagedCopy(*cache, torch.tensor([4199], device=dev, dtype=torch.int32), torch.tensor([4150], device=dev, dtype=torch.int32))
    table = torch.tensor([[4198, 4150]], dtype=torch.int32, device=dev)
    assert blockedAttention.pagedKeep(*cache, table, torch.tensor([255], device=dev), torch.tensor([[1, 7]], device=dev)).tolist() == [257]
    for i, c in enumerate(cache):
        assert (c[4150] == 3 + i).all() and (c[4198, :, 255] == 3 + i).all() and (c[4198, :, 200] == 7 + i).all()
        assert c.count_nonzero() == 2 * c[0].numel() + 2 * heads * dim


def test_versions_tell_of_the_writes(dev):
    cache = make_cache(dev, torch.float16, 3, 2, 4, 8)
    was = [c._version for c in cache]
    blockedAttention.pagedCopy(*cache, torch.tensor([0], device=dev, dtype=torch.int32), torch.tensor([1], device=dev, dtype=torch.int32))
    assert all(c._version > w for c, w in zip(cache, was))


def test_keep_in_a_graph(dev):
    cache = make_cache(dev, torch.float16, 6, 2, 8, 64)
    table = torch.tensor([[2, 4], [1, 0]], dtype=torch.int32, device=dev)
    base, path = torch.tensor([3, 0], device=dev), torch.tensor([[1, 4, 5], [2, -1, -1]], device=dev)
    blockedAttention.pagedKeep(*cache, table, base, path)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lens = blockedAttention.pagedKeep(*cache, table, base, path)
    for paths in ([[0, 2, 7], [3, 4, 5]], [[-1, -1, -1], [0, 6, 7]], [[1, 2, 3], [1, 2, 3]]):
        path.copy_(torch.tensor(paths))
        want, n = expect_keep([c.cpu() for c in cache], table.cpu(), [3, 0], paths, 8)
        graph.replay()
        torch.cuda.synchronize()
        assert lens.tolist() == n
        for c, w in zip(cache, want):
            assert torch.equal(bits(c).cpu(), w)


def test_entry_points_take_a_cache_without_scales(dev):
    cache = make_cache(dev, FP8, 3, 2, 4, 16)
    c = capi.paged_cache(*cache)
    want = bits(cache[0])[1].clone()
    capi.paged_copy(c, torch.tensor([1], device=dev, dtype=torch.int32), torch.tensor([0], device=dev, dtype=torch.int32))
    assert torch.equal(bits(cache[0])[0], want)
