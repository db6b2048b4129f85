"""pagedTreeAttention against the same in 64 bits on the CPU.

Bound, per value, as for pagedAttention: |o - ref| <= u |ref| + (u + 2 e + (n + 64) 2^-24 + 2^-20) (P |V|) + 2^-24, with
u = 2^-11 (fp16) or 2^-8 (bf16), half the spacing of the type's numbers, for one rounding of the result and one of each
probability, e = (dim + 8) 2^-24 max_t |scale| sum_d |q_d k_td| for a score's products and sum in fp32 (an error of e in a
score moves a probability and the sum it is divided by by a factor of at most 1 +- e each), n + 64 additions of probabilities
in fp32, 2^-20 for the exponential; the last term is the smallest step of fp16.
Everything in the cache that no row sees is NaN.
"""
import pytest
import torch

import blockedAttention
from blockedattention_amd import capi

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


class Drafts:
    """Requests with drafts in pages of a cache, on the CPU, and the result in 64 bits with its bound.

    base, nodes: tokens before the draft and nodes of each request; mask: "tree", "chain" (none is passed), "any" (random bits, some
    rows none).  pad rows belong to no request.
    """

    room = 0                                                  # tokens that a row of the table has room for at least

    def __init__(self, base, nodes, heads, group, dim, page, dtype=torch.float16, fp8=False, mask="tree", order="heads", seed=0, spread=2.0,
                 pad=0, front=0, extra=2, words=None):
        g = torch.Generator().manual_seed(seed)
        self.base, self.nodes, self.heads, self.group, self.dim, self.page, self.dtype, self.fp8 = base, nodes, heads, group, dim, page, dtype, fp8
        lens = [b + n for b, n in zip(base, nodes)]
        self.lens = lens
        need = [-(-n // page) for n in lens]
        pages, width = sum(need) + extra, max(max(need + [1]) + 1, -(-self.room // page))
        self.table = torch.full((len(lens), width), -1, dtype=torch.int32)
        numbers, at = torch.randperm(pages, generator=g, dtype=torch.int32), 0
        shape = (pages, heads, page, dim) if order == "heads" else (pages, page, heads, dim)
        store = FP8 if fp8 else dtype
        kv = [torch.full(shape, float("nan"), dtype=dtype).to(store) for _ in range(2)]
        self.k, self.v = (c if order == "heads" else c.transpose(1, 2) for c in kv)
        self.scales = [0.01 * (1 + torch.rand(heads, generator=g)) for _ in range(2)] if fp8 else [None, None]
        for r, n in enumerate(lens):
            self.table[r, :need[r]] = numbers[at:at + need[r]]
            at += need[r]
            for c in (self.k, self.v):
                x = torch.randn((heads, n, dim), generator=g)
                self.put(c, r, 0, (x * 100).clamp(-448, 448).to(FP8) if fp8 else x.to(dtype))
        self.accum = [front]
        for n in nodes:
            self.accum.append(self.accum[-1] + n)
        self.tokens = self.accum[-1] + pad
        self.q = (torch.randn((heads * group, self.tokens, dim), generator=g) * spread).to(dtype)
        most = max(nodes + [1])
        words = words or -(-most // 64)
        self.sees = []                                        # [nodes, nodes] of each request
        for n in nodes:
            s = torch.zeros((n, n), dtype=torch.bool)
            for i in range(n):
                if mask == "chain":
                    s[i, :i + 1] = True
                elif mask == "tree":
                    p = int(torch.randint(-1, i, (1,), generator=g)) if i else -1
                    if p >= 0:
                        s[i] = s[p]
                    s[i, i] = True
                elif torch.rand(1, generator=g) > 0.2:
                    s[i] = torch.rand(n, generator=g) < 0.5
            self.sees.append(s)
        self.mask = None
        if mask != "chain":
            bits = torch.zeros((self.tokens, words * 64), dtype=torch.bool)
            bits[:front] = True
            bits[self.accum[-1]:] = True
            for s, a, n in zip(self.sees, self.accum, nodes):
                bits[a:a + n, :n] = s
                bits[a:a + n, n:] = torch.rand((n, words * 64 - n), generator=g) < 0.5          # bits of nodes that are not there
            self.mask = (bits.reshape(self.tokens, words, 64).long() << torch.arange(64)).sum(-1)

    def put(self, cache, r, first, x):
        """Tokens first .. of a request, [heads, tokens, dim]."""
        raw, mine = (cache.view(torch.uint8), x.view(torch.uint8)) if self.fp8 else (cache, x)
        for i in range(x.shape[1]):
            t = first + i
            raw[int(self.table[r, t // self.page]), :, t % self.page] = mine[:, i]

    def values(self, cache, scale, r, n):
        """[heads, tokens, dim] in 64 bits."""
        pages = self.table[r, :-(-n // self.page)].long()
        c = cache.view(torch.uint8)[pages].view(FP8) if self.fp8 else cache[pages]
        x = c.to(torch.float32).double().transpose(0, 1).reshape(self.heads, -1, self.dim)[:, :n]
        return x * scale.double()[:, None, None] if self.fp8 else x

    def seen(self, r, window):
        n, base = self.nodes[r], self.base[r]
        s = torch.cat([torch.ones((n, base), dtype=torch.bool), self.sees[r]], 1)
        if window:
            s &= s.flip(1).cumsum(1).flip(1) <= window
        return s

    def expect(self, scale, window=0):
        out = torch.zeros(self.q.shape, dtype=torch.float64)
        bound = torch.zeros_like(out)
        u = U[self.dtype]
        for r, n in enumerate(self.lens):
            a, nodes = self.accum[r], self.nodes[r]
            if nodes == 0:
                continue
            k, v = self.values(self.k, self.scales[0], r, n), self.values(self.v, self.scales[1], r, n)
            q = self.q[:, a:a + nodes].double().reshape(self.heads, self.group, nodes, self.dim)
            s = self.seen(r, window)
            kq = torch.where(s, torch.matmul(q, k[:, None].transpose(2, 3)) * scale, -torch.inf)
            top = kq.amax(-1, keepdim=True)
            p = torch.exp(kq - torch.where(top == -torch.inf, 0.0, top))
            p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
            some = s.any(0)                                   # what no row sees may be NaN
            v = torch.where(some[:, None], v, 0.0)[:, None]
            size = torch.matmul(q.abs(), k[:, None].abs().transpose(2, 3))
            e = (self.dim + 8) * 2.0 ** -24 * abs(scale) * torch.where(s, size, 0.0).amax(-1, keepdim=True)
            o = torch.matmul(p, v)
            b = u * o.abs() + (u + 2 * e + (n + 64) * 2.0 ** -24 + 2.0 ** -20) * torch.matmul(p, v.abs()) + 2.0 ** -24
            out[:, a:a + nodes], bound[:, a:a + nodes] = o.reshape(-1, nodes, self.dim), b.reshape(-1, nodes, self.dim)
        return out, bound

    def operands(self, dev):
        on = lambda x: None if x is None else x.to(dev)  # noqa: E731
        if not hasattr(self, "there"):
            order = self.k.stride(1) < self.k.stride(2)
            move = lambda c: c.transpose(1, 2).contiguous().to(dev).transpose(1, 2) if order else c.to(dev)  # noqa: E731
            self.there = dict(kCache=move(self.k), vCache=move(self.v), table=on(self.table), lens=torch.tensor(self.lens, device=dev, dtype=torch.int64),
                              accum=torch.tensor(self.accum, device=dev), mask=on(self.mask), kScale=on(self.scales[0]), vScale=on(self.scales[1]))
        return self.there

    def run(self, dev, scale, window=0, flat=False):
        q = self.q.reshape(self.q.shape[0], -1).to(dev) if flat else self.q.transpose(0, 1).contiguous().to(dev).transpose(0, 1)
        out = blockedAttention.pagedTreeAttention(q, **self.operands(dev), scale=scale, window=window)
        assert out.shape == q.shape and out.dtype == q.dtype and out.stride() == q.stride()
        return out.reshape(self.q.shape)

    def check(self, dev, scale=None, window=0, flat=False):
        scale = self.dim ** -0.5 if scale is None else scale
        ref, bound = self.expect(scale, window)
        got = self.run(dev, scale, window, flat).double().cpu()
        bad = ~((got - ref).abs() <= bound)
        assert not bad.any(), (int(bad.sum()), bad.nonzero()[:5].tolist(), (got - ref).abs()[bad].max().item())
        return got


@pytest.mark.parametrize("dtype,fp8", [(torch.float16, False), (torch.bfloat16, False), (torch.float16, True), (torch.bfloat16, True)])
@pytest.mark.parametrize("mask", ["tree", "chain", "any"])
@pytest.mark.parametrize("dim,page,order", [(128, 16, "heads"), (64, 16, "tokens"), (80, 24, "heads"), (100, 7, "tokens"), (256, 32, "heads")])
def test_types_masks_dimensions(dev, dtype, fp8, mask, dim, page, order):
    Drafts([0, 1, 33, 200, 5, 64], [3, 1, 17, 30, 0, 8], 2, 4, dim, page, dtype, fp8, mask, order, pad=3, front=2).check(dev)


@pytest.mark.parametrize("dim", [1, 2, 3, 4, 7, 8, 9, 15, 16, 24, 31, 32, 33, 40, 48, 63, 65, 72, 96, 104, 127, 129, 136, 160, 192, 200, 224, 250, 255])
@pytest.mark.parametrize("fp8", [False, True])
def test_every_kind_of_dimension(dev, dim, fp8):
    Drafts([50, 0, 130], [9, 5, 20], 2, 2, dim, 16, torch.float16, fp8, seed=dim).check(dev, 0.7 * dim ** -0.5, flat=dim % 2 == 0)


@pytest.mark.parametrize("group,nodes", [(1, 1), (1, 31), (1, 33), (1, 128), (1, 129), (3, 11), (4, 8), (4, 32), (4, 33), (5, 7), (8, 16), (8, 50), (16, 64), (32, 5), (33, 3),
                                         (100, 2), (1, 300)])
def test_rows_of_a_key_head(dev, group, nodes):
    """One row to several blocks of rows."""
    Drafts([70, 3], [nodes, max(1, nodes // 2)], 2, group, 64, 16, torch.bfloat16, seed=nodes).check(dev)
    Drafts([70, 3], [nodes, max(1, nodes // 2)], 1, group, 128, 16, torch.float16, mask="chain", seed=nodes).check(dev)


@pytest.mark.parametrize("page", [1, 2, 3, 5, 8, 12, 17, 32, 48, 64, 100, 256, 1000])
def test_pages(dev, page):
    Drafts([0, 10, 63, 64, 300], [5, 7, 2, 40, 9], 2, 3, 64, page, torch.float16, seed=page).check(dev)


@pytest.mark.parametrize("window", [1, 2, 5, 31, 32, 33, 64, 100, 199, 1000])
@pytest.mark.parametrize("mask", ["tree", "chain", "any"])
def test_windows(dev, window, mask):
    Drafts([0, 10, 200, 301], [70, 7, 20, 130], 2, 2, 64, 16, torch.bfloat16, mask=mask, seed=window).check(dev, window=window)


@pytest.mark.parametrize("words", [1, 2, 5])
def test_masks_narrower_and_wider_than_the_draft(dev, words):
    b = Drafts([40, 9], [100, 20], 1, 2, 64, 16, mask="any", words=5, seed=words)
    b.mask = b.mask[:, :words].contiguous() if words == 2 else b.mask[:, :words]
    for s in b.sees:
        s[:, 64 * words:] = False
    b.check(dev)


def test_rows_that_see_nothing(dev):
    """Drafts without tokens before them whose rows have no bits: zeros, and zeros for padded rows."""
    b = Drafts([0, 0, 4], [6, 70, 3], 2, 3, 64, 16, mask="any", pad=5, front=1)
    for r, rows in ((0, range(6)), (1, (0, 5, 69))):
        for i in rows:
            b.sees[r][i] = False
            b.mask[b.accum[r] + i] = 0
    b.sees[0][2, 1] = True
    b.mask[b.accum[0] + 2, 0] = 2
    got = b.check(dev)
    assert (got[:, 1:3] == 0).all() and (got[:, 4:7] == 0).all() and (got[:, 0] == 0).all() and (got[:, -5:] == 0).all()
    assert (got[:, 3] != 0).any()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("value", ["nan", "inf", "-inf"])
def test_what_a_row_does_not_see_has_no_influence(dev, value, fp8):
    """Keys and values of nodes that some rows see and others do not: those others stay as they are."""
    if fp8 and value != "nan":
        pytest.skip("e4m3 has no infinities")
    b = Drafts([37, 0], [40, 9], 2, 2, 64, 16, torch.float16, fp8, mask="any", seed=8)
    ref, bound = b.expect(0.125)
    x = torch.full((2, 1, 64), float(value), dtype=torch.float16)
    x = x.to(FP8) if fp8 else x
    for r, node in ((0, 3), (0, 21), (1, 0)):
        for c in (b.k, b.v):
            b.put(c, r, b.base[r] + node, x)
    got = b.run(dev, 0.125).double().cpu()
    for r in range(2):
        a = b.accum[r]
        for i in range(b.nodes[r]):
            touched = any(b.sees[r][i, n] for q, n in ((0, 3), (0, 21), (1, 0)) if q == r)
            mine = got[:, a + i]
            if not touched:
                assert ((mine - ref[:, a + i]).abs() <= bound[:, a + i]).all(), (r, i)
            elif value == "nan":
                assert mine.isnan().all()


def test_infinite_values_that_are_seen(dev):
    b = Drafts([5, 33], [20, 3], 1, 2, 64, 16, torch.float16, mask="any", seed=2)
    v = torch.zeros((1, 1, 64), dtype=torch.float16)
    v[..., 7], v[..., 9], v[..., 20] = torch.inf, -torch.inf, torch.nan
    b.put(b.v, 0, 5 + 11, v)
    w = torch.zeros((1, 1, 64), dtype=torch.float16)
    w[..., 7], w[..., 9] = torch.inf, torch.inf
    b.put(b.v, 0, 5 + 4, w)
    got = b.run(dev, 0.125).double().cpu()
    for i in range(20):
        x, y = bool(b.sees[0][i, 11]), bool(b.sees[0][i, 4])
        row = got[:, i]
        assert (row[:, 7] == torch.inf).all() if x or y else row[:, 7].isfinite().all()
        assert (row[:, 9].isnan().all() if x and y else (row[:, 9] == (-torch.inf if x else torch.inf)).all()) if x or y else row[:, 9].isfinite().all()
        assert row[:, 20].isnan().all() if x else row[:, 20].isfinite().all()
        assert row[:, 30:].isfinite().all()


def test_scores_far_from_zero(dev):
    """Scores of up to 2^27, where neighbouring numbers of fp32 lie 8 apart: the largest one takes all."""
    for dtype in (torch.float16, torch.bfloat16):
        b = Drafts([300], [5], 1, 2, 64, 16, dtype, spread=30.0, seed=3)
        for scale in (2.0 ** 12, 2.0 ** 16, 2.0 ** 19, -2.0 ** 16):
            got = b.run(dev, scale).double().cpu()
            k, v = b.values(b.k, None, 0, 305), b.values(b.v, None, 0, 305)
            q = b.q.double().reshape(1, 2, 5, 64)
            s = torch.where(b.seen(0, 0), torch.matmul(q, k[:, None].transpose(2, 3)) * scale, -torch.inf)
            want = v[0][s.argmax(-1)].reshape(2, 5, 64)
            lead = s.topk(2, -1).values
            clear = (lead[..., 0] - lead[..., 1] > 2.0 ** -18 * lead[..., 0].abs() + 40).reshape(2, 5)       # by more than a score's error
            assert clear.sum() >= 7 and got.isfinite().all()
            assert ((got - want).abs() <= U[dtype] * 2 * want.abs() + 1e-6)[clear].all()


def test_one_long_request_is_split_and_joined(dev):
    for lens, nodes, heads, group in (([30000], [3], 1, 1), ([9000, 20, 700], [40, 1, 9], 2, 4), ([5000] * 2, [64, 33], 1, 8)):
        for fp8 in (False, True):
            Drafts(lens, nodes, heads, group, 128, 16, torch.bfloat16, fp8, seed=nodes[0]).check(dev)
    Drafts([6000], [7], 2, 2, 256, 24, torch.float16).check(dev)


def test_many_requests(dev):
    g = torch.Generator().manual_seed(0)
    base = torch.randint(0, 90, (700,), generator=g).tolist()
    nodes = torch.randint(0, 6, (700,), generator=g).tolist()
    Drafts(base, nodes, 1, 2, 64, 16, torch.float16, pad=9).check(dev)
    Drafts(base[:300], nodes[:300], 3, 1, 32, 8, torch.bfloat16, mask="chain").check(dev, window=20)


def test_agrees_with_one_query_a_request(dev):
    """Drafts of a token are what pagedAttention answers."""
    b = Drafts([0, 4, 100, 900], [1, 1, 1, 1], 2, 4, 128, 16, torch.float16, mask="chain", seed=6)
    o = b.operands(dev)
    q = b.q.to(dev)
    one = blockedAttention.pagedAttention(q, o["kCache"], o["vCache"], o["table"], o["lens"], scale=0.1, window=77)
    ref, bound = b.expect(0.1, 77)
    for got in (one, blockedAttention.pagedTreeAttention(q, **o, scale=0.1, window=77)):
        assert ((got.double().cpu() - ref).abs() <= bound).all()


def test_page_numbers_outside_the_cache(dev):
    b = Drafts([40, 40, 40], [4, 4, 4], 1, 2, 64, 16, torch.float16, mask="chain")
    ref, bound = b.expect(0.125)
    for bad in (-1, b.k.shape[0], (1 << 31) - 1, -(1 << 31)):
        table = b.operands(dev)["table"].clone()
        table[1, 0] = bad
        got = blockedAttention.pagedTreeAttention(b.q.to(dev), **{**b.operands(dev), "table": table}, scale=0.125).double().cpu()
        assert got[:, 4:8].isnan().all()
        for rows in (slice(0, 4), slice(8, 12)):
            assert ((got[:, rows] - ref[:, rows]).abs() <= bound[:, rows]).all()
        # behind the window nobody looks at it
        got = blockedAttention.pagedTreeAttention(b.q.to(dev), **{**b.operands(dev), "table": table}, scale=0.125, window=8).double().cpu()
        ref8, bound8 = b.expect(0.125, 8)
        assert ((got - ref8).abs() <= bound8).all()


def test_tokens_beyond_the_row_do_not_exist(dev):
    """A length that the table's row does not hold, and one shorter than the draft."""
    b = Drafts([40], [6], 1, 2, 64, 16, torch.float16, mask="chain")
    o = b.operands(dev)
    got = blockedAttention.pagedTreeAttention(b.q.to(dev), **{**o, "table": o["table"][:, :2].contiguous()}, scale=0.125).double().cpu()
    short = Drafts([40], [6], 1, 2, 64, 16, torch.float16, mask="chain")
    short.sees[0][:] = False
    k, v = (short.values(c, None, 0, 46)[:, :32] for c in (b.k, b.v))
    p = torch.softmax(torch.matmul(b.q.double().reshape(1, 2, 6, 64), k[:, None].transpose(2, 3)) * 0.125, -1)
    want = torch.matmul(p, v[:, None]).reshape(2, 6, 64)
    assert ((got - want).abs() <= 2 ** -9 * torch.matmul(p, v[:, None].abs()).reshape(2, 6, 64) + 1e-6).all()
    # of a window only tokens that exist
    got = blockedAttention.pagedTreeAttention(b.q.to(dev), **{**o, "table": o["table"][:, :2].contiguous()}, scale=0.125, window=5).double().cpu()
    p = torch.softmax(torch.matmul(b.q.double().reshape(1, 2, 6, 64), k[:, None, 27:].transpose(2, 3)) * 0.125, -1)
    want = torch.matmul(p, v[:, None, 27:]).reshape(2, 6, 64)
    assert ((got - want).abs() <= 2 ** -9 * torch.matmul(p, v[:, None, 27:].abs()).reshape(2, 6, 64) + 1e-6).all()
    got = blockedAttention.pagedTreeAttention(b.q.to(dev), **{**o, "lens": o["lens"] * 0 + 3}, scale=0.125)      # nodes 0 .. 2 are there
    k, v = (b.values(c, None, 0, 3) for c in (b.k, b.v))
    s = torch.where(torch.arange(3) <= torch.arange(6)[:, None], torch.matmul(b.q.double().reshape(1, 2, 6, 64), k[:, None].transpose(2, 3)) * 0.125, -torch.inf)
    want = torch.matmul(torch.softmax(s, -1), v[:, None]).reshape(2, 6, 64)
    assert ((got.double().cpu() - want).abs() <= 2 ** -9 * want.abs().amax() + 1e-6).all()
    for n in (0, -5, -(1 << 62)):
        assert (blockedAttention.pagedTreeAttention(b.q.to(dev), **{**o, "lens": o["lens"] * 0 + n}, scale=0.125) == 0).all()


def test_layouts(dev):
    """Caches and queries that are parts of larger arrays, rows at odd addresses, one table row for all requests."""
    b = Drafts([50, 21, 0], [9, 4, 6], 2, 2, 64, 16, torch.float16, pad=2)
    ref, bound = b.expect(0.125)
    o = b.operands(dev)
    for dim_pad, shift in ((8, 0), (3, 1), (64, 8)):
        wide = [torch.full((*c.shape[:3], 64 + dim_pad + shift), float("nan"), dtype=c.dtype, device=dev) for c in (b.k, b.v)]
        parts = [w[..., shift:shift + 64] for w in wide]
        for p, c in zip(parts, (o["kCache"], o["vCache"])):
            p.copy_(c)
        qw = torch.zeros((b.tokens, 4, 64 + dim_pad + shift), dtype=torch.float16, device=dev)[..., shift:shift + 64].transpose(0, 1)
        qw.copy_(b.q)
        got = blockedAttention.pagedTreeAttention(qw, **{**o, "kCache": parts[0], "vCache": parts[1]}, scale=0.125)
        assert ((got.double().cpu() - ref).abs() <= bound).all()
        assert all(w[..., :shift].isnan().all() and w[..., shift + 64:].isnan().all() for w in wide)
    wide_mask = torch.full((b.tokens, 7), -1, dtype=torch.int64, device=dev)
    wide_mask[:, :1] = o["mask"]
    got = blockedAttention.pagedTreeAttention(b.q.to(dev), **{**o, "mask": wide_mask[:, :1]}, scale=0.125)
    assert ((got.double().cpu() - ref).abs() <= bound).all()
    # one row of the table for all: requests of the same tokens
    c = Drafts([44, 44], [4, 4], 2, 2, 64, 16, torch.float16, mask="chain")
    for cache in (c.k, c.v):
        x = c.values(cache, None, 0, 48).half()
        c.put(cache, 1, 0, x)
    ref, bound = c.expect(0.125)
    p = c.operands(dev)
    got = blockedAttention.pagedTreeAttention(c.q.to(dev), **{**p, "table": p["table"][:1].expand(2, -1)}, scale=0.125)
    assert ((got.double().cpu() - ref).abs() <= bound).all()


def test_nothing_to_do(dev):
    b = Drafts([5], [3], 1, 2, 64, 16, torch.float16, mask="chain")
    o = b.operands(dev)
    none = dict(o, table=o["table"][:0], lens=o["lens"][:0], accum=o["accum"][:1])
    assert (blockedAttention.pagedTreeAttention(b.q.to(dev), **none) == 0).all()
    assert blockedAttention.pagedTreeAttention(b.q[:, :0].to(dev), **o).shape == (2, 0, 64)
    empty = dict(o, kCache=o["kCache"][:0], vCache=o["vCache"][:0])
    assert blockedAttention.pagedTreeAttention(b.q.to(dev), **empty).isnan().all()
    assert (blockedAttention.pagedTreeAttention(b.q.to(dev), **dict(empty, lens=o["lens"] * 0)) == 0).all()


def test_sums_that_do_not_fit_the_rows(dev):
    """Sums beyond the rows, or that go down: rows inside are written, no other memory is."""
    b = Drafts([50, 21, 4], [9, 4, 6], 2, 2, 64, 16, torch.float16, mask="chain")
    o = b.operands(dev)
    ref, bound = b.expect(0.125)
    whole = torch.full((4, 60, 64), 7.0, dtype=torch.float16, device=dev)
    out = whole[:, 20:39]
    cache = capi.paged_cache(o["kCache"], o["vCache"])
    for sums in ([0, 9, 13, 19 + (1 << 40)], [0, 9, 13, -5], [-(1 << 50), 9, 13, 19], [0, 9, 3, 19], [0, 1 << 62, 13, 19], [5, 5, 5, 5]):
        capi.paged_tree_attention(cache, b.q.to(dev), o["table"], o["lens"], torch.tensor(sums, device=dev), out, None, 0.125)
        assert (whole[:, :20] == 7).all() and (whole[:, 39:] == 7).all()
    capi.paged_tree_attention(cache, b.q.to(dev), o["table"], o["lens"], o["accum"], out, None, 0.125)
    assert ((out.double().cpu() - ref).abs() <= bound).all()


def test_offsets_past_32_bits(dev):
    """Pages whose byte offsets pass 2^32; the pages between are never touched."""
    pages, page, dim = 40000, 64, 256
    k, v = (torch.empty((pages, 2, page, dim), dtype=torch.bfloat16, device=dev) for _ in range(2))
    b = Drafts([500, 70], [20, 9], 2, 2, dim, page, torch.bfloat16)
    o = b.operands(dev)
    n = b.k.shape[0]
    k[pages - n:], v[pages - n:] = o["kCache"], o["vCache"]
    table = torch.where(o["table"] >= 0, o["table"] + pages - n, -1).int()
    ref, bound = b.expect(0.0625)
    got = blockedAttention.pagedTreeAttention(b.q.to(dev), **{**o, "kCache": k, "vCache": v, "table": table}, scale=0.0625)
    assert ((got.double().cpu() - ref).abs() <= bound).all()


def test_streams_and_graph_replays(dev):
    """Calls whose requests are split between workgroups, on several streams and replayed beside each other."""
    batches = [Drafts([3000, 900], [12, 40], 2, 2, 64, 16, torch.float16, seed=1), Drafts([2500] * 3, [9, 1, 30], 1, 4, 128, 16, torch.bfloat16, seed=2),
               Drafts([40] * 50, [3] * 50, 2, 2, 64, 16, torch.bfloat16, seed=3)]
    qs = [b.q.to(dev) for b in batches]
    call = lambda i: blockedAttention.pagedTreeAttention(qs[i], **batches[i].operands(dev), scale=0.125)  # noqa: E731
    want = [call(i) for i in range(3)]
    for b, w in zip(batches, want):
        ref, bound = b.expect(0.125)
        assert ((w.double().cpu() - ref).abs() <= bound).all()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], [[] for _ in range(3)]
    for _ in range(12):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(i))
    torch.cuda.synchronize()
    assert all(torch.equal(x, w) for w, g in zip(want, got) for x in g)
    graphs, outs = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(i))
        graphs.append(graph)
    for step in range(4):
        for i in range(2):                                    # other queries each time
            qs[i].copy_(batches[i].q.to(dev) * (1 + step))
        now = [call(i) for i in range(2)]
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, n) for o, n in zip(outs, now)), step


def test_counters_are_zero_after_every_call(dev):
    counters = capi.paged_counters(dev)
    for b in (Drafts([3000, 900], [12, 40], 2, 2, 64, 16, seed=1), Drafts([20000], [3], 1, 1, 128, 16, seed=2)):
        o = b.operands(dev)
        out = torch.full_like(b.q, 5.0).to(dev)
        for _ in range(2):
            capi.paged_tree_attention(capi.paged_cache(o["kCache"], o["vCache"]), b.q.to(dev), o["table"], o["lens"], o["accum"], out, o["mask"], 0.125, 0, counters)
            assert (counters == 0).all()
        ref, bound = b.expect(0.125)
        assert ((out.double().cpu() - ref).abs() <= bound).all()


@pytest.mark.parametrize("scale", [-0.3, 0.0, -0.0, 1e-39])
@pytest.mark.parametrize("nodes", [5, 12, 40])
def test_scales_of_either_sign_and_none(dev, scale, nodes):
    for dtype, dim, fp8 in ((torch.float16, 64, False), (torch.bfloat16, 128, True), (torch.float16, 84, False), (torch.bfloat16, 7, False)):
        Drafts([0, 100, 30], [nodes, nodes, 1], 2, 2, dim, 16, dtype, fp8, seed=nodes).check(dev, scale)


def test_scores_far_from_zero_for_many_rows(dev):
    for dtype in (torch.float16, torch.bfloat16):
        b = Drafts([300], [40], 1, 4, 64, 16, dtype, spread=30.0, seed=3)
        for scale in (2.0 ** 12, 2.0 ** 19, -2.0 ** 16):
            got = b.run(dev, scale).double().cpu()
            k, v = b.values(b.k, None, 0, 340), b.values(b.v, None, 0, 340)
            q = b.q.double().reshape(1, 4, 40, 64)
            s = torch.where(b.seen(0, 0), torch.matmul(q, k[:, None].transpose(2, 3)) * scale, -torch.inf)
            want = v[0][s.argmax(-1)].reshape(4, 40, 64)
            lead = s.topk(2, -1).values
            clear = (lead[..., 0] - lead[..., 1] > 2.0 ** -18 * lead[..., 0].abs() + 40).reshape(4, 40)
            assert clear.sum() >= 100 and got.isfinite().all()
            assert ((got - want).abs() <= U[dtype] * 2 * want.abs() + 1e-6)[clear].all()


@pytest.mark.parametrize("nodes", [3, 8, 40])
def test_many_small_probabilities(dev, nodes):
    """60000 tokens of 2^-21 beside one of 1, which have to count in the sum as they do in the result.

    Bound: 2^-10 for a probability as a denormal number of fp16 (2^-15 in steps of 2^-24 after lifting, half a step), 2^-11 for the result, and 2000
    additions in fp32, a step each, twice."""
    b = Drafts([60000], [nodes], 1, 4, 16, 64, torch.float16)
    b.k[torch.isfinite(b.k)] = 0.0
    b.v[torch.isfinite(b.v)] = 1.0
    b.k[int(b.table[0, 0]), 0, 0, 0] = 21.0
    b.v[int(b.table[0, 0]), 0, 0] = 0.0
    b.q.zero_()
    b.q[..., 0] = 1.0
    got = b.run(dev, 0.6931471805599453).double().cpu()
    n = 60000 - 1 + b.seen(0, 0)[:, 60000:].sum(-1).double()
    want = (n * 2.0 ** -21 / (1 + n * 2.0 ** -21))[None, :, None]
    assert ((got - want).abs() <= (2.0 ** -10 + 2.0 ** -11 + 4000 * 2.0 ** -24) * want).all()


@pytest.fixture
def roomy(monkeypatch):
    """Tables of long rows: calls with many rows then have units of 64 or 128 of them, however few the tokens are."""
    monkeypatch.setattr(Drafts, "room", 4096)


@pytest.mark.parametrize("dtype,fp8", [(torch.float16, False), (torch.bfloat16, False), (torch.float16, True), (torch.bfloat16, True)])
@pytest.mark.parametrize("mask", ["tree", "chain", "any"])
@pytest.mark.parametrize("dim,page,order", [(128, 16, "heads"), (64, 16, "tokens"), (80, 24, "heads"), (100, 7, "tokens"), (256, 32, "heads")])
def test_many_rows(dev, roomy, dtype, fp8, mask, dim, page, order):
    Drafts([0, 1, 33, 200, 5, 64], [3, 40, 80, 30, 0, 8], 2, 4, dim, page, dtype, fp8, mask, order, pad=3, front=2).check(dev)
    if dim <= 64:
        Drafts([0, 1, 33, 200, 5, 64], [3, 20, 17, 30, 0, 8], 2, 4, dim, page, dtype, fp8, mask, order, pad=3, front=2).check(dev)


@pytest.mark.parametrize("dim", [1, 2, 3, 4, 7, 8, 9, 15, 16, 24, 31, 32, 33, 40, 48, 63, 65, 72, 96, 104, 127, 129, 136, 160, 192, 200, 224, 250, 255])
@pytest.mark.parametrize("fp8", [False, True])
def test_many_rows_of_every_kind_of_dimension(dev, roomy, dim, fp8):
    Drafts([50, 0, 130], [30, 15, 60], 2, 2, dim, 16, torch.float16, fp8, seed=dim).check(dev, 0.7 * dim ** -0.5, flat=dim % 2 == 0)
    if dim <= 64:
        Drafts([50, 0, 130], [30, 15, 20], 2, 2, dim, 16, torch.float16, fp8, seed=dim).check(dev, 0.7 * dim ** -0.5)


@pytest.mark.parametrize("window", [1, 33, 64, 199, 1000])
@pytest.mark.parametrize("mask", ["tree", "chain", "any"])
def test_windows_of_many_rows(dev, window, mask):
    Drafts([0, 10, 200, 301], [70, 7, 20, 130], 4, 16, 64, 16, torch.bfloat16, mask=mask, seed=window).check(dev, window=window)


@pytest.mark.parametrize("page", [1, 3, 17, 64, 100, 1000])
def test_pages_of_many_rows(dev, roomy, page):
    Drafts([0, 10, 63, 64, 300], [25, 17, 42, 40, 29], 2, 3, 64, page, torch.float16, seed=page).check(dev)


def test_unusual_values_in_long_tables(dev, roomy):
    """Many rows over values that are not finite, rows that see nothing, scales of either sign."""
    test_rows_that_see_nothing(dev)
    for value in ("nan", "inf", "-inf"):
        test_what_a_row_does_not_see_has_no_influence(dev, value, False)
    test_what_a_row_does_not_see_has_no_influence(dev, "nan", True)
    test_scores_far_from_zero_for_many_rows(dev)
    for scale in (-0.3, 0.0, 1e-39):
        test_scales_of_either_sign_and_none(dev, scale, 40)
    for words in (1, 2, 5):
        test_masks_narrower_and_wider_than_the_draft(dev, words)


@pytest.mark.parametrize("dim,fp8", [(64, False), (128, True), (256, False), (100, False)])
def test_infinite_values_that_many_rows_see(dev, roomy, dim, fp8):
    b = Drafts([5, 33], [60, 3], 1, 4, dim, 16, torch.float16, fp8, mask="any", seed=2)
    v = torch.zeros((1, 1, dim), dtype=torch.float16)
    v[..., 7], v[..., 20] = torch.nan if fp8 else torch.inf, torch.nan
    b.put(b.v, 0, 5 + 11, v.to(FP8) if fp8 else v)
    got = b.run(dev, 0.125).double().cpu()
    for i in range(60):
        x, row = bool(b.sees[0][i, 11]), got[:, i]
        assert (row[:, 7].isnan() if fp8 else row[:, 7] == torch.inf).all() if x else row[:, 7].isfinite().all()
        assert row[:, 20].isnan().all() if x else row[:, 20].isfinite().all()
        assert row[:, 30:].isfinite().all()


@pytest.mark.parametrize("dim,fp8", [(64, False), (128, True), (256, False), (100, False), (7, False)])
def test_page_numbers_outside_the_cache_for_many_rows(dev, roomy, dim, fp8):
    b = Drafts([40, 40, 40], [40, 40, 40], 1, 2, dim, 16, torch.float16, fp8, mask="chain")
    ref, bound = b.expect(0.125)
    for bad in (-1, b.k.shape[0], (1 << 31) - 1, -(1 << 31)):
        table = b.operands(dev)["table"].clone()
        table[1, 0] = bad
        got = blockedAttention.pagedTreeAttention(b.q.to(dev), **{**b.operands(dev), "table": table}, scale=0.125).double().cpu()
        assert got[:, 40:80].isnan().all()
        for rows in (slice(0, 40), slice(80, 120)):
            assert ((got[:, rows] - ref[:, rows]).abs() <= bound[:, rows]).all()


@pytest.mark.parametrize("nodes", [3, 8, 40])
def test_scales_that_are_no_numbers(dev, roomy, nodes):
    """A head whose keys have a scale of NaN: its rows are NaN, the other's are not."""
    b = Drafts([100], [nodes], 2, 4, 128, 16, torch.bfloat16, True, seed=nodes)
    b.scales[0][1] = float("nan")
    got = b.run(dev, 0.1)
    assert got[:4].isfinite().all() and got[4:].isnan().all()
    assert b.run(dev, float("nan")).isnan().all()


@pytest.mark.parametrize("dim,fp8", [(256, False), (160, True), (131, False)])
def test_many_rows_of_many_dimensions_in_small_units(dev, dim, fp8):
    """Few requests over few tokens, more rows than a unit has; the same in long tables."""
    for room in (0, 4096):
        Drafts.room = room
        try:
            Drafts([60, 0, 300], [40, 70, 1], 2, 4, dim, 16, torch.bfloat16, fp8, mask="tree", seed=dim, pad=2).check(dev, window=0 if dim == 256 else 90)
        finally:
            Drafts.room = 0
