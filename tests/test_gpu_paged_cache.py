"""pagedResize against a list for the stack, pagedAppend against the rounding in 64 bits: whole numbers and stored
values have to be equal."""
import math

import numpy as np
import pytest
import torch

import blockedAttention
from blockedattention_amd import capi

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn


# ------------------------------------------------------------------ pagedResize
class Model:
    """What pagedResize does, request by request."""

    def __init__(self, requests, page, width, pool, seed=0):
        rng = np.random.default_rng(seed)
        self.page, self.width = page, width
        self.stack = [int(x) for x in rng.permutation(pool)]
        self.free = list(self.stack)
        self.table = np.full((requests, width), -1, dtype=np.int32)
        self.lens = [0] * requests
        self.verdict = 0

    def pages(self, n):
        return -(-n // self.page)

    def step(self, new, tokens):
        count, verdict = len(self.stack), self.verdict
        most = self.page * self.width
        take = sum(max(self.pages(n) - self.pages(o), 0) for o, n in zip(self.lens, new))
        drop = sum(max(self.pages(o) - self.pages(n), 0) for o, n in zip(self.lens, new))
        if any(n < 0 for n in new):
            verdict |= 4
        if any(n > most for n in new):
            verdict |= 2
        if not verdict:
            verdict |= (1 if take > count + drop else 0) | (8 if sum(max(n - o, 0) for o, n in zip(self.lens, new)) > tokens else 0)
        self.verdict = verdict
        if verdict:
            return [-1] * tokens, [0] * (len(new) + 1), list(self.lens)
        given = [int(self.table[r, c]) for r, (o, n) in enumerate(zip(self.lens, new)) for c in range(self.pages(n), self.pages(o))]
        self.stack += given[::-1]
        slots, accum = [], [0]
        for r, (o, n) in enumerate(zip(self.lens, new)):
            for c in range(self.pages(o), self.pages(n)):
                self.table[r, c] = self.stack.pop()
            slots += [int(self.table[r, t // self.page]) * self.page + t % self.page for t in range(o, n)]
            accum.append(len(slots))
        self.free[count:len(self.stack)] = self.stack[count:]
        self.lens = list(new)
        return slots + [-1] * (tokens - len(slots)), accum, list(self.lens)


class Device:
    def __init__(self, m, dev, stride=0):
        self.dev, self.page = dev, m.page
        wide = torch.from_numpy(np.concatenate([m.table, np.full((len(m.lens), stride), -7, np.int32)], 1)).to(dev)
        self.wide, self.table = wide, wide[:, :m.width]
        self.free = torch.tensor(m.free, dtype=torch.int32, device=dev)
        self.state = torch.tensor([len(m.stack), 0], device=dev)
        self.lens = torch.tensor(m.lens, dtype=torch.int64, device=dev)

    def step(self, new, tokens):
        args = (self.table, self.free, self.state, self.lens, torch.tensor(new, dtype=torch.int64, device=self.dev), self.page, tokens)
        first = blockedAttention.pagedResize(*args)
        slots, accum, lens, state = blockedAttention.pagedResize(*args)      # the same call again writes the same
        for a, b in zip(first, (slots, accum, lens, state)):
            assert torch.equal(a, b)
        self.lens, self.state = lens, state
        return slots, accum


def same(m, d, new, tokens):
    slots, accum, lens = m.step(new, tokens)
    got = d.step(new, tokens)
    assert got[0].tolist() == slots
    assert got[1].tolist() == accum
    assert d.lens.tolist() == lens
    assert d.state.tolist() == [len(m.stack), m.verdict]
    assert np.array_equal(d.table.cpu().numpy(), m.table)
    assert d.free.tolist() == m.free
    assert (d.wide[:, m.width:] == -7).all()


@pytest.mark.parametrize("requests", [1, 2, 63, 64, 65, 300, 1025, 5000])
@pytest.mark.parametrize("page", [1, 3, 16, 64])
def test_many_steps(dev, requests, page):
    rng = np.random.default_rng(requests + page)
    width = 7
    m = Model(requests, page, width, requests * width, seed=page)
    d = Device(m, dev, stride=page % 2)
    for step in range(8):
        kind = rng.integers(0, 5, requests)
        old = np.array(m.lens)
        new = np.select([kind == 0, kind == 1, kind == 2, kind == 3],
                        [old + 1, old, 0 * old, rng.integers(0, page * width + 1, requests)], np.maximum(old - rng.integers(0, 2 * page + 1, requests), 0))
        new = np.minimum(new, page * width) if step != 5 else 0 * new       # everything ends once
        grow = int(np.maximum(new - old, 0).sum())
        same(m, d, [int(x) for x in new], grow + step % 3)


def test_growing_and_shrinking_back_leaves_the_stack(dev):
    m = Model(40, 16, 9, 40 * 9, seed=1)
    d = Device(m, dev)
    rng = np.random.default_rng(0)
    base = [int(x) for x in rng.integers(0, 100, 40)]
    same(m, d, base, sum(base))
    free, count = d.free.clone(), d.state[0].item()
    up = [x + int(y) for x, y in zip(base, rng.integers(0, 44, 40))]
    same(m, d, up, sum(up) - sum(base))
    same(m, d, base, 0)
    assert torch.equal(d.free, free) and d.state[0].item() == count


def test_long_prompts(dev):
    m = Model(5, 16, 4000, 10000, seed=2)
    d = Device(m, dev)
    same(m, d, [0, 63999, 1, 20000, 7777], 63999 + 1 + 20000 + 7777)
    same(m, d, [30000, 16, 2, 0, 64000], 30000 + 1 + 64000 - 7777 + 11)


@pytest.mark.parametrize("new,tokens,verdict", [
    ([33, 16, 0], 60, 1),            # three + one + nothing of three free pages
    ([161, 0, 0], 200, 2),           # eleven pages in a row of ten
    ([-1, 5, 0], 60, 4),
    ([17, 16, 0], 32, 8),            # 33 new tokens
    ([161, 16, -5], 200, 6),
])
def test_verdicts_change_nothing_and_stay(dev, new, tokens, verdict):
    m = Model(3, 16, 10, 3, seed=3)
    d = Device(m, dev)
    same(m, d, new, tokens)
    assert d.state[1].item() == verdict
    same(m, d, [1, 1, 1], 3)         # refused too: the verdict stays until the program looks at it
    assert d.state[1].item() == verdict
    m.verdict = 0
    d.state = torch.tensor([d.state[0].item(), 0], device=dev)
    same(m, d, [1, 1, 1], 3)
    assert d.state.tolist() == [0, 0]


def test_states_and_lengths_that_cannot_be(dev):
    m = Model(2, 16, 4, 6, seed=4)
    for state, lens, verdict in (([-1, 0], [0, 0], 16), ([6, 0], [64, 0], 16), ([2, 0], [65, 0], 4), ([2, 0], [-3, 0], 4)):
        d = Device(m, dev)
        d.state, d.lens = torch.tensor(state, device=dev), torch.tensor(lens, device=dev)
        before = d.table.clone(), d.free.clone()
        slots, accum = d.step([0, 1], 5)
        assert d.state.tolist() == [state[0], verdict]
        assert slots.tolist() == [-1] * 5 and accum.tolist() == [0, 0, 0] and d.lens.tolist() == lens
        assert torch.equal(d.table, before[0]) and torch.equal(d.free, before[1])


def test_no_requests_and_no_tokens(dev):
    e = lambda *s, dt=torch.int64: torch.zeros(s, dtype=dt, device=dev)  # noqa: E731
    slots, accum, lens, state = blockedAttention.pagedResize(e(0, 4, dt=torch.int32), e(3, dt=torch.int32), torch.tensor([3, 0], device=dev),
                                                             e(0), e(0), 16, 2)
    assert slots.tolist() == [-1, -1] and accum.tolist() == [0] and lens.numel() == 0 and state.tolist() == [3, 0]
    slots, accum, lens, state = blockedAttention.pagedResize(e(2, 0, dt=torch.int32), e(0, dt=torch.int32), torch.tensor([0, 0], device=dev),
                                                             e(2), e(2), 16, 0)
    assert slots.numel() == 0 and accum.tolist() == [0, 0, 0] and state.tolist() == [0, 0]


def test_resize_under_graph_capture(dev):
    m = Model(70, 16, 6, 500, seed=5)
    d = Device(m, dev)
    new = torch.zeros(70, dtype=torch.int64, device=dev)
    blockedAttention.pagedResize(d.table, d.free, d.state, d.lens, new, 16, 90)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        slots, accum, lens, state = blockedAttention.pagedResize(d.table, d.free, d.state, d.lens, new, 16, 90)
    rng = np.random.default_rng(1)
    for _ in range(4):
        want = [max(0, min(96, n + int(x))) for n, x in zip(m.lens, rng.integers(-3, 2, 70))]
        new.copy_(torch.tensor(want))
        graph.replay()
        torch.cuda.synchronize()
        expect = m.step(want, 90)
        assert slots.tolist() == expect[0] and accum.tolist() == expect[1] and lens.tolist() == expect[2]
        assert state.tolist() == [len(m.stack), m.verdict] and np.array_equal(d.table.cpu().numpy(), m.table) and d.free.tolist() == m.free
        d.lens.copy_(lens); d.state.copy_(state)


def test_resize_refusals(dev):
    m = Model(3, 16, 10, 9)
    d = Device(m, dev)
    call = blockedAttention.pagedResize
    good = dict(table=d.table, free=d.free, state=d.state, lens=d.lens, newLens=d.lens, pageSize=16, tokens=4)
    for name, value, text in (("table", d.table.long(), "int32"), ("table", d.table.cpu(), "GPU tensor"), ("table", d.table.t(), "contiguous"),
                              ("free", d.free.long(), "int32"), ("state", d.state[:1], "state must be"), ("state", d.state.int(), "int64"),
                              ("lens", d.lens[:2], "lens must be"), ("newLens", d.lens.int(), "int64"), ("pageSize", 0, "at least one"),
                              ("tokens", -1, "negative")):
        with pytest.raises(RuntimeError, match=text):
            call(**{**good, name: value})


# ------------------------------------------------------------------ pagedAppend
def e4m3(x):
    """Nearest e4m3 value, ties to even, of numbers in 64 bits."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def bits(t):
    return t.view(torch.uint8 if t.dtype == FP8 else torch.int16)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads,dim,page,tokens", [(1, 1, 1, 1), (2, 8, 16, 5), (3, 64, 16, 100), (8, 128, 16, 64), (5, 37, 24, 41),
                                                   (2, 80, 32, 300), (1, 256, 64, 33), (4, 20, 8, 70), (32, 96, 16, 9), (2, 129, 3, 17)])
@pytest.mark.parametrize("order,flat", [("heads", True), ("tokens", False)])
def test_append(dev, dtype, fp8, heads, dim, page, tokens, order, flat):
    g = torch.Generator().manual_seed(heads * dim + tokens)
    pages = -(-tokens // page) + 3
    shape = (pages, heads, page, dim) if order == "heads" else (pages, page, heads, dim)
    store = FP8 if fp8 else dtype
    caches = [torch.randn(shape, generator=g).to(dtype).to(store) for _ in range(2)]
    caches = [c if order == "heads" else c.transpose(1, 2) for c in caches]
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    skip = torch.randperm(tokens, generator=g)[:tokens // 5]
    slots[skip[::2]] = -1
    slots[skip[1::2]] = pages * page + 5
    rows = [(torch.randn((tokens, heads, dim), generator=g) * 3).to(dtype).transpose(0, 1) for _ in range(2)]
    scales = [torch.rand(heads, generator=g) * 0.05 + 0.001 for _ in range(2)] if fp8 else [None, None]
    want = []
    for x, c, s in zip(rows, caches, scales):
        w = c.float() if fp8 else c.clone()
        for t in range(tokens):
            if 0 <= slots[t] < pages * page:
                y = x[:, t]
                if fp8:
                    y = e4m3((y.float() / s[:, None]).double()).float()
                w[slots[t] // page, :, slots[t] % page] = y
        want.append(w.to(store))
    on = [c.transpose(1, 2).to(dev).transpose(1, 2) if order == "tokens" else c.to(dev) for c in caches]
    k, v = ((x.reshape(heads, -1) if flat else x).to(dev) for x in rows)
    versions = [c._version for c in on]
    blockedAttention.pagedAppend(k, v, *on, slots.to(dev), *(None if s is None else s.to(dev) for s in scales))
    for c, w, before in zip(on, want, versions):
        assert torch.equal(bits(c.contiguous().cpu()), bits(w.contiguous()))
        assert c._version > before


def test_append_limits_ties_and_what_is_no_number(dev):
    x = torch.tensor([448., 449., 464., 1e4, -1e4, float("inf"), float("-inf"), float("nan"), 0., -0., 17., 19., 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, 1.0625])
    x = torch.cat([x, torch.zeros(16)]).reshape(1, 2, 16)
    cache = [torch.zeros((1, 1, 4, 16), device=dev, dtype=FP8) for _ in range(2)]
    one = torch.ones(1, device=dev)
    blockedAttention.pagedAppend(x.bfloat16().to(dev), x.bfloat16().to(dev), *cache, torch.tensor([2, 0], device=dev), one, one)
    want = torch.tensor([448., 448., 448., 448., -448., 448., -448., float("nan"), 0., -0., 16., 20., 2.0 ** -9, 0., 2.0 ** -8, 1.0])
    got = cache[0][0, 0, 2].float().cpu()
    assert torch.equal(torch.nan_to_num(got, nan=999.), torch.nan_to_num(want, nan=999.))
    assert torch.equal(torch.signbit(got[8:10]), torch.tensor([False, True]))
    assert (bits(cache[1][0, 0, 1:2].contiguous()) == 0).all() and (bits(cache[1][0, 0, 3:].contiguous()) == 0).all()


def test_append_beyond_2_31_elements(dev):
    cache = [torch.empty((140000, 2, 64, 128), dtype=torch.float16, device=dev) for _ in range(2)]
    x = torch.randn((2, 70, 128), device=dev).half()
    slots = 140000 * 64 - 1 - 3 * torch.arange(70, device=dev)
    blockedAttention.pagedAppend(x, 2 * x, *cache, slots)
    for c, y in zip(cache, (x, 2 * x)):
        assert torch.equal(c[slots // 64, :, slots % 64], y.transpose(0, 1))


def test_append_of_views_at_any_alignment(dev):
    x = torch.randn((9, 3, 70), device=dev).half()
    cache = [torch.zeros((2, 3, 8, 67), dtype=torch.float16, device=dev)[..., 1:65] for _ in range(2)]
    slots = torch.arange(9, device=dev)
    blockedAttention.pagedAppend(x[..., 3:67].transpose(0, 1), x[..., 4:68].transpose(0, 1), *cache, slots)
    for c, y in zip(cache, (x[..., 3:67], x[..., 4:68])):
        assert torch.equal(c[slots // 8, :, slots % 8], y)
    one = torch.randn((1, 64), device=dev).half()                         # the same token everywhere: strides of zero
    same = one.expand(3, 5, 64)
    blockedAttention.pagedAppend(same, same, *cache, slots[:5] + 9)
    assert (cache[0][1, :, 1:6] == one).all() and (cache[0][1, :, 0] == x[8, :, 3:67]).all()


def test_append_refusals_and_nothing_to_do(dev):
    cache = [torch.zeros((2, 3, 8, 64), dtype=torch.float16, device=dev) for _ in range(2)]
    x, slots = torch.ones((3, 4, 64), dtype=torch.float16, device=dev), torch.arange(4, device=dev)
    call = blockedAttention.pagedAppend
    call(x[:, :0], x[:, :0], *cache, slots[:0])
    call(x, x, cache[0][:0], cache[1][:0], slots)
    assert all((c == 0).all() for c in cache)
    ones = torch.ones(3, device=dev)
    for bad, text in ((lambda: call(x[:2], x[:2], *cache, slots), "3 heads"), (lambda: call(x, x[:, :3], *cache, slots), "number of tokens"),
                      (lambda: call(x.bfloat16(), x.bfloat16(), *cache, slots), "cache's dtype"), (lambda: call(x, x.bfloat16(), *cache, slots), "same dtype"),
                      (lambda: call(x, x, *cache, slots[:3]), "slots must be"), (lambda: call(x, x, *cache, slots.int()), "int64"),
                      (lambda: call(x[..., :32], x[..., :32], *cache, slots), "rows of 64"), (lambda: call(x, x, *cache, slots, ones, ones), "belong to"),
                      (lambda: call(x, x, *(c.to(FP8) for c in cache), slots), "needs kScale"), (lambda: call(x.cpu(), x, *cache, slots), "GPU tensor"),
                      (lambda: call(x.clone().requires_grad_(), x, *cache, slots), "no backward pass")):
        with pytest.raises(RuntimeError, match=text):
            bad()


def test_c_abi_gives_the_operators_results(dev):
    m = Model(4, 16, 5, 30, seed=6)
    d, e = Device(m, dev), Device(m, dev)
    new = torch.tensor([17, 0, 40, 3], device=dev)
    want = blockedAttention.pagedResize(d.table, d.free, d.state, d.lens, new, 16, 64)
    got = [torch.full_like(t, 99) for t in want]
    capi.paged_resize(e.table, e.free, e.state, e.lens, new, 16, *got)
    assert all(torch.equal(a, b) for a, b in zip(want, got)) and torch.equal(d.table, e.table) and torch.equal(d.free, e.free)
    caches = [torch.zeros((30, 2, 16, 64), dtype=torch.bfloat16, device=dev) for _ in range(4)]
    x = torch.randn((2, 64, 64), device=dev).bfloat16()
    blockedAttention.pagedAppend(x, -x, *caches[:2], want[0])
    capi.paged_append(capi.paged_cache(*caches[2:]), x, -x, want[0])
    assert torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3]) and caches[0].abs().sum() > 0
    assert math.isclose(caches[0].float().abs().sum().item(), x[:, :60].float().abs().sum().item(), rel_tol=1e-6)
