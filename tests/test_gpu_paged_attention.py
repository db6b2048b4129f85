"""pagedAttention against the same in 64 bits on the CPU.

Bound, per value: |o - ref| <= u |ref| + (u + 2 e + (n + 64) 2^-24 + 2^-20) (P |V|) + 2^-24, with u = 2^-11 (fp16) or 2^-8
(bf16), half the spacing of the type's numbers, for one rounding of the result and one of each probability,
e = (dim + 8) 2^-24 max_t |scale| sum_d |q_d k_td| for a score's products and sum in fp32 (an error of e in a score moves a
probability and the sum it is divided by by a factor of at most 1 +- e each), n + 64 additions of probabilities in fp32,
2^-20 for the exponential; the last term is the smallest step of fp16.
Everything in the cache that no request sees is NaN.
"""
import numpy as np
import pytest
import torch

import blockedAttention
from blockedattention_amd import capi

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


class Batch:
    """Requests of the given lengths in pages of a cache, on the CPU, and the result in 64 bits with its bound."""

    def __init__(self, lens, heads, group, dim, page, dtype=torch.float16, fp8=False, order="heads", seed=0, spread=2.0, extra=2):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.group, self.dtype, self.page, self.dim, self.fp8 = list(lens), group, dtype, page, dim, fp8
        need = [-(-n // page) for n in lens]
        pages = sum(need) + extra
        width = max(need + [1]) + 1
        self.table = torch.full((len(lens), width), -1, dtype=torch.int32)
        order_of = torch.randperm(pages, generator=g, dtype=torch.int32)
        at, kv = 0, []
        shape = (pages, heads, page, dim) if order == "heads" else (pages, page, heads, dim)
        store = FP8 if fp8 else dtype
        for _ in range(2):
            c = torch.full(shape, float("nan"), dtype=dtype).to(store)
            kv.append(c if order == "heads" else c.transpose(1, 2))
        self.k, self.v = kv
        self.scales = [0.01 * (1 + torch.rand(heads, generator=g)) for _ in range(2)] if fp8 else [None, None]
        for r, n in enumerate(lens):
            self.table[r, :need[r]] = order_of[at:at + need[r]]
            at += need[r]
            for c in (self.k, self.v):
                x = torch.randn((heads, n, dim), generator=g)
                x = (x * 100).clamp(-448, 448).to(FP8) if fp8 else x.to(dtype)
                raw, mine = (c.view(torch.uint8), x.view(torch.uint8)) if fp8 else (c, x)
                for i in range(need[r]):
                    rows = mine[:, i * page:(i + 1) * page]
                    raw[int(self.table[r, i]), :, :rows.shape[1]] = rows
        self.q = (torch.randn((heads * group, len(lens), dim), generator=g) * spread).to(dtype)
        self.heads = heads

    def tokens(self, cache, scale, r, first, n):
        """[heads, tokens, dim] in 64 bits."""
        pages = self.table[r, :-(-n // self.page)].long()
        c = cache.view(torch.uint8)[pages].view(FP8) if self.fp8 else cache[pages]
        x = c.to(torch.float32).double().transpose(0, 1).reshape(self.heads, -1, self.dim)[:, first:n]
        return x * scale.double()[:, None, None] if self.fp8 else x

    def expect(self, scale, window=0):
        out = torch.zeros(self.q.shape, dtype=torch.float64)
        bound = torch.zeros_like(out)
        u = U[self.dtype]
        for r, n in enumerate(self.lens):
            if n == 0:
                continue
            first = max(0, n - window) if window else 0
            k, v = self.tokens(self.k, self.scales[0], r, first, n), self.tokens(self.v, self.scales[1], r, first, n)
            q = self.q[:, r].double().reshape(self.heads, self.group, self.dim)
            p = torch.softmax(torch.matmul(q, k.transpose(1, 2)) * scale, -1)
            e = (self.dim + 8) * 2.0 ** -24 * abs(scale) * torch.matmul(q.abs(), k.abs().transpose(1, 2)).amax(-1, keepdim=True)
            o = torch.matmul(p, v)
            b = u * o.abs() + (u + 2 * e + (n + 64) * 2.0 ** -24 + 2.0 ** -20) * torch.matmul(p, v.abs()) + 2.0 ** -24
            out[:, r], bound[:, r] = o.reshape(-1, self.dim), b.reshape(-1, self.dim)
        return out, bound

    def run(self, dev, scale, window=0, flat=False):
        q = self.q.reshape(self.q.shape[0], -1) if flat else self.q.transpose(0, 1).contiguous().to(dev).transpose(0, 1)
        ks, vs = (None if s is None else s.to(dev) for s in self.scales)
        put = lambda c: c.transpose(1, 2).to(dev).transpose(1, 2) if c.stride(1) < c.stride(2) else c.to(dev)  # noqa: E731
        out = blockedAttention.pagedAttention(q.to(dev), put(self.k), put(self.v), self.table.to(dev), torch.tensor(self.lens).to(dev),
                                              scale=scale, window=window, kScale=ks, vScale=vs)
        assert out.shape == q.shape and out.dtype == self.dtype
        return out.reshape(self.q.shape)

    def check(self, dev, scale=None, window=0, flat=False):
        scale = self.dim ** -0.5 if scale is None else scale
        got = self.run(dev, scale, window, flat).double().cpu()
        ref, bound = self.expect(scale, window)
        assert not torch.isnan(got).any(), "NaN from what no request sees"
        over = ((got - ref).abs() - bound).max().item()
        assert over <= 0, f"off by {over} more than the bound"
        return got


LENS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 0, 127, 128, 129, 200, 333]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dim", [8, 32, 64, 80, 96, 128, 192, 256])
def test_dimensions(dev, dtype, fp8, dim):
    Batch(LENS, 2, 4, dim, 16, dtype, fp8, seed=dim).check(dev)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dim", [1, 7, 20, 37, 66, 100, 129, 250])
@pytest.mark.parametrize("order", ["heads", "tokens"])
def test_rows_at_any_alignment(dev, fp8, dim, order):
    Batch([5, 0, 40, 129, 1], 3, 2, dim, 16, torch.bfloat16, fp8, order, seed=dim).check(dev, flat=True)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dim", [3, 8, 9, 15, 16, 17, 33, 64, 65, 119, 128, 200, 255])
@pytest.mark.parametrize("page,group,window", [(16, 3, 0), (24, 32, 40), (7, 1, 0), (64, 32, 0)])
def test_rows_between_nan(dev, fp8, dim, page, group, window):
    """Rows an odd number of elements apart; what lies between them is NaN."""
    b = Batch([1, 0, 33, 700, 64], 2, group, dim, page, torch.float16, fp8, seed=dim + page)
    ref, bound = b.expect(0.25, window)
    caches = []
    for c in (b.k, b.v):
        wide = torch.full((*c.shape[:3], dim + 2 + dim % 2 + 1), float("nan"), dtype=b.dtype).to(c.dtype)
        raw, mine = (wide.view(torch.uint8), c.view(torch.uint8)) if fp8 else (wide, c)
        raw[..., 1:dim + 1] = mine
        caches.append(wide.to(dev)[..., 1:dim + 1])
    scales = [None if x is None else x.to(dev) for x in b.scales]
    got = blockedAttention.pagedAttention(b.q.to(dev), *caches, b.table.to(dev), torch.tensor(b.lens).to(dev), 0.25, window, *scales)
    assert ((got.double().cpu() - ref).abs() <= bound).all()


@pytest.mark.parametrize("page", [1, 2, 7, 8, 16, 24, 32, 48, 64, 100, 256])
@pytest.mark.parametrize("order", ["heads", "tokens"])
@pytest.mark.parametrize("fp8", [False, True])
def test_pages(dev, page, order, fp8):
    Batch(LENS, 2, 4, 64, page, torch.float16, fp8, order, seed=page).check(dev)
    Batch([1, 500, 77], 1, 8, 128, page, torch.bfloat16, fp8, order, seed=page + 1).check(dev, flat=True)


@pytest.mark.parametrize("group", [1, 2, 3, 5, 8, 15, 16, 17, 32, 71])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_shared_heads(dev, group, dim):
    Batch([70, 0, 1, 290], 2, group, dim, 16, torch.bfloat16, seed=group).check(dev)


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 31, 33, 100, 128, 300, 5000])
@pytest.mark.parametrize("page", [16, 24, 64])
def test_window(dev, window, page):
    Batch(LENS, 2, 2, 64, page, torch.float16, seed=window).check(dev, window=window)


@pytest.mark.parametrize("lens", [[20000], [9000, 1, 0, 4000], [3000] * 5 + [40] * 30, [1] * 700, [0, 0, 0], [130] * 257])
@pytest.mark.parametrize("fp8", [False, True])
def test_work_split_over_the_length(dev, lens, fp8):
    Batch(lens, 2, 4, 64, 32, torch.float16, fp8, seed=len(lens)).check(dev)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1.0, 4.0])
def test_scales_of_either_sign_and_none(dev, scale):
    for dtype in (torch.float16, torch.bfloat16):
        Batch([1, 50, 300, 700], 2, 4, 64, 16, dtype, spread=1.0, seed=9).check(dev, scale=scale)


def test_a_few_keys_far_above_thousands(dev):
    """Probabilities far below the largest still count in their sum: one key stands out by 12, 8000 are alike."""
    b = Batch([8001], 1, 2, 64, 16, torch.float16, seed=4)
    b.q[:] = 0; b.q[:, :, 0] = 1.0
    for c in (b.k,):
        flat = torch.zeros((8001, 64), dtype=torch.float16); flat[4000, 0] = 12.0
        for i in range(-(-8001 // 16)):
            rows = flat[i * 16:(i + 1) * 16]
            c[int(b.table[0, i]), 0, :len(rows)] = rows
    b.check(dev, scale=1.0)


def test_infinities_and_nan_count_only_where_they_are_seen(dev):
    b = Batch([100, 40, 64, 9], 1, 2, 64, 16, torch.float16, seed=6)
    at = lambda r, t: (int(b.table[r, t // 16]), 0, t % 16)  # noqa: E731
    b.v[at(0, 50)][3] = float("inf")              # one column of request 0
    b.k[at(1, 7)][5] = float("nan")               # all of request 1
    for t in range(9):
        b.k[at(3, t)][:] = float("inf")           # scores of both signs or NaN: as the softmax of them
    got = b.run(dev, 0.125).double().cpu()
    ref, _ = b.expect(0.125)
    assert not torch.isfinite(got[:, 0, 3]).any()
    assert torch.isnan(got[:, 1]).all()
    keep = torch.ones(64, dtype=torch.bool); keep[3] = False
    assert (got[:, 0, keep] - ref[:, 0, keep]).abs().max() < 2e-2 and (got[:, 2] - ref[:, 2]).abs().max() < 2e-2
    assert torch.isnan(ref[:, 3]).all() and torch.isnan(got[:, 3]).all()


def test_keys_at_the_lowest_value(dev):
    """Scores of minus infinity for every token are what the softmax makes of them, for some tokens they are zeros."""
    b = Batch([48, 48], 1, 1, 32, 16, torch.bfloat16, seed=7)
    b.q[:] = 1.0
    for r, count in ((0, 48), (1, 47)):
        for t in range(count):
            b.k[int(b.table[r, t // 16]), 0, t % 16] = float("-inf")
    got = b.run(dev, 1.0).double().cpu()
    assert torch.isnan(got[:, 0]).all()
    last = b.v[int(b.table[1, 2]), 0, 15].double()
    assert torch.equal(got[0, 1], last)


def test_page_numbers_outside_the_cache_are_not_read(dev):
    b = Batch([40, 40, 40], 2, 2, 64, 16, torch.float16, seed=8)
    ref, bound = b.expect(0.125)
    for bad in (-1, b.k.shape[0], 2 ** 31 - 1):
        b.table[1, 1] = bad
        got = b.run(dev, 0.125).double().cpu()
        assert torch.isnan(got[:, 1]).all()
        assert ((got - ref).abs() <= bound)[:, [0, 2]].all()


def test_lengths_beyond_the_table_and_below_zero(dev):
    b = Batch([48, 5], 1, 1, 64, 16, torch.float16, seed=8)
    table = b.table[:, :3].contiguous().to(dev)
    call = lambda lens: blockedAttention.pagedAttention(b.q.to(dev), b.k.to(dev), b.v.to(dev), table, torch.tensor(lens).to(dev), 0.125)  # noqa: E731
    assert torch.equal(call([2 ** 40, 5]), call([48, 5]))
    got = call([48, -3])
    assert (got[:, 1] == 0).all() and not (got[:, 0] == 0).all()


def test_a_cache_beyond_2_31_elements(dev):
    page, heads, dim, pages = 64, 2, 128, 140000                          # 2.3e9 elements an array
    k = torch.empty((pages, heads, page, dim), dtype=torch.float16, device=dev)
    v = torch.empty_like(k)
    b = Batch([200, 90], heads, 4, dim, page, torch.float16, seed=11)
    ref, bound = b.expect(0.1)
    table = torch.full_like(b.table, -1)
    for r, n in enumerate(b.lens):
        for i in range(-(-n // page)):
            table[r, i] = pages - 1 - 7 * i - 100 * r
            k[int(table[r, i])] = b.k[int(b.table[r, i])].to(dev)
            v[int(table[r, i])] = b.v[int(b.table[r, i])].to(dev)
    got = blockedAttention.pagedAttention(b.q.to(dev), k, v, table.to(dev), torch.tensor(b.lens).to(dev), 0.1)
    assert ((got.double().cpu() - ref).abs() <= bound).all()


def test_other_orders_of_a_cache_and_offset_views(dev):
    b = Batch([100, 33], 3, 2, 64, 16, torch.float16, seed=12)
    ref, bound = b.expect(0.125)
    lens, table = torch.tensor(b.lens).to(dev), b.table.to(dev)
    k, v, q = b.k.to(dev), b.v.to(dev), b.q.to(dev)
    head_first = [c.transpose(0, 1).contiguous().transpose(0, 1) for c in (k, v)]                  # [heads][pages][page][dim]
    one = torch.stack([k, v], 1)                                                                   # keys and values by turns
    odd = [torch.nn.functional.pad(c, (1, 2))[..., 1:65] for c in (k, v)]                    # rows off any alignment
    wide = torch.zeros((2, 50), dtype=torch.int32, device=dev); wide[:, 7:7 + table.size(1)] = table
    for kc, vc, tb in ((*head_first, table), (one[:, 0], one[:, 1], table), (*odd, table), (k, head_first[1], wide[:, 7:7 + table.size(1)])):
        got = blockedAttention.pagedAttention(q, kc, vc, tb, lens, 0.125)
        assert ((got.double().cpu() - ref).abs() <= bound).all()
    odd_q = torch.nn.functional.pad(q, (1, 0))[..., 1:]
    got = blockedAttention.pagedAttention(odd_q, k, v, table, lens, 0.125)
    assert ((got.double().cpu() - ref).abs() <= bound).all()


def test_the_same_call_gives_the_same_bits_and_needs_no_other_stream(dev):
    b = Batch([3000, 70, 900, 0, 1], 4, 4, 128, 16, torch.bfloat16, seed=13)
    first = b.check(dev).to(torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [b.run(dev, 128 ** -0.5) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    for t in again:
        assert torch.equal(t.cpu(), first)


def test_under_graph_capture(dev):
    b = Batch([3000, 70, 900, 0], 2, 4, 64, 16, torch.float16, seed=14)
    q, k, v, table = b.q.to(dev), b.k.to(dev), b.v.to(dev), b.table.to(dev)
    lens = torch.tensor(b.lens).to(dev)
    want = blockedAttention.pagedAttention(q, k, v, table, lens, 0.125)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = blockedAttention.pagedAttention(q, k, v, table, lens, 0.125)
    for n in (b.lens, [100, 70, 1, 0], [3000, 0, 900, 0], b.lens):
        lens.copy_(torch.tensor(n))
        graph.replay()
        torch.cuda.synchronize()
        want = blockedAttention.pagedAttention(q, k, v, table, lens, 0.125)
        assert torch.equal(out, want), n


def test_c_abi_gives_the_operator_s_result(dev):
    b = Batch([300, 70, 0], 2, 4, 64, 16, torch.float16, True, seed=15)
    k, v, (ks, vs) = b.k.to(dev), b.v.to(dev), (s.to(dev) for s in b.scales)
    cache = capi.paged_cache(k, v, ks, vs)
    q, lens, table = b.q.to(dev), torch.tensor(b.lens).to(dev), b.table.to(dev)
    out = torch.full_like(q, float("nan"))
    capi.paged_attention(cache, q, table, lens, out, 0.125)
    assert torch.equal(out, blockedAttention.pagedAttention(q, k, v, table, lens, 0.125, 0, ks, vs))


def test_empty_batches_and_refusals(dev):
    b = Batch([30, 5], 2, 2, 64, 16, torch.float16, seed=1)
    q, k, v, table, lens = b.q.to(dev), b.k.to(dev), b.v.to(dev), b.table.to(dev), torch.tensor(b.lens).to(dev)
    call = blockedAttention.pagedAttention
    assert call(q[:, :0], k, v, table[:0], lens[:0]).shape == (4, 0, 64)
    assert (call(q, k, v, table[:, :0], lens) == 0).all()                 # rows without pages: no tokens
    assert (call(q, k[:0], v[:0], table, 0 * lens) == 0).all()            # a cache without pages
    for bad, text in (
            (lambda: call(q[:3], k, v, table, lens), "multiple of the cache's"),
            (lambda: call(q.float(), k, v, table, lens), "fp16 or bf16"),
            (lambda: call(q.bfloat16(), k, v, table, lens), "cache's dtype"),
            (lambda: call(q[..., :60], k, v, table, lens), "rows of 64"),
            (lambda: call(q, k, v[:, :1], table, lens), "both be"),
            (lambda: call(q, k, v.bfloat16(), table, lens), "same dtype"),
            (lambda: call(q, k.float(), v.float(), table, lens), "holds fp16"),
            (lambda: call(q, k, v, table.long(), lens), "int32"),
            (lambda: call(q, k, v, table[:1], lens), "q has 2 rows"),
            (lambda: call(q, k, v, table, lens.int()), "int64"),
            (lambda: call(q, k, v, table, lens[:1]), "lens must be"),
            (lambda: call(q, k, v, table, lens.cpu()), "GPU tensor"),
            (lambda: call(q, k, v, table, lens, window=-1), "window"),
            (lambda: call(q, k.transpose(2, 3), v.transpose(2, 3), table, lens), "contiguous"),
            (lambda: call(q, k, v, table, lens, kScale=torch.ones(2, device=dev)), "belong to"),
            (lambda: call(q, k.to(FP8), v.to(FP8), table, lens), "needs kScale"),
            (lambda: call(q, k.to(FP8), v.to(FP8), table, lens, kScale=torch.ones(3, device=dev), vScale=torch.ones(2, device=dev)), "one entry per head"),
            (lambda: call(q.clone().requires_grad_(), k, v, table, lens), "no backward pass"),
            (lambda: call(torch.zeros((2, 2, 300), device=dev, dtype=torch.float16), torch.zeros((1, 2, 1, 300), device=dev, dtype=torch.float16),
                          torch.zeros((1, 2, 1, 300), device=dev, dtype=torch.float16), table, lens), "1 to 256")):
        with pytest.raises(RuntimeError, match=text):
            bad()
