"""The paged cache's operators where a count passes what a launch or 32 bits hold at once."""
import pytest
import torch

import blockedAttention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("order", ["heads", "tokens"])
def test_append_of_more_tokens_than_a_grid_dimension_holds_workgroups(dev, order):
    """2^24 + 5 tokens of 257 heads (heads of a token together: a workgroup a token), nearly all of them padding."""
    heads, dim, page, tokens = 257, 8, 4, (1 << 24) + 5
    shape = (3, page, heads, dim) if order == "tokens" else (3, heads, page, dim)
    cache = [torch.zeros(shape, dtype=torch.float16, device=dev) for _ in range(2)]
    cache = [c.transpose(1, 2) if order == "tokens" else c for c in cache]
    g = torch.Generator().manual_seed(0)
    x = torch.randn((heads, 1, dim), generator=g).half().to(dev)
    slots = torch.full((tokens,), -1, dtype=torch.int64, device=dev)
    at = torch.tensor([0, 1, (1 << 20) - 1, 1 << 20, (1 << 23) + 7, (1 << 24) - 1, 1 << 24, tokens - 1], device=dev)
    slots[at] = torch.tensor([3, 11, 0, 5, 7, 10, 2, 8], device=dev)
    blockedAttention.pagedAppend(x.expand(heads, tokens, dim), -x.expand(heads, tokens, dim), *cache, slots)
    there = torch.zeros(12, dtype=torch.bool, device=dev)
    there[slots[at]] = True
    for c, sign in zip(cache, (1, -1)):
        want = torch.where(there.view(3, 1, page, 1), sign * x[None].expand(3, heads, page, dim), 0)
        assert torch.equal(c, want)


@pytest.mark.parametrize("page,width", [(4202512, 511), (9216668, 233), (6487866, 331)])
def test_attention_over_nearly_2_31_tokens(dev, page, width):
    """Requests of 2^31 - 16 (pages of a multiple of 16 tokens), 2^31 - 4 (of 4) and 2^31 - 2 tokens, and of three less.

    Every column but the last is page 0, whose keys are 0 and whose values are 1, so a query of 0 sees equal probabilities: sums of
    powers of two, exact in fp32 but for the joining of parts and the quotient; the result is rounded once to fp16 (2^-11).
    The other query finds its token at the very end, 86 powers of two above the rest.  What is behind is NaN.
    """
    dim, most = 8, page * width
    assert (1 << 31) - 32 < most < 1 << 31
    k = torch.zeros((3, 1, page, dim), dtype=torch.float16, device=dev)
    v = torch.ones_like(k)
    g = torch.Generator().manual_seed(width)
    last = torch.randn((2, 200, dim), generator=g).half().to(dev)
    for i, end in ((1, page), (2, page - 3)):
        v[i] = 3.0
        v[i, 0, end - 200:end] = last[i - 1]
        k[i, 0, end - 1, 0] = 60.0
        k[i, 0, end:] = float("nan")
        v[i, 0, end:] = float("nan")
    table = torch.zeros((3, width), dtype=torch.int32, device=dev)
    table[0, -1], table[1, -1] = 1, 2
    lens = torch.tensor([most, most - 3, 40], device=dev)
    q = torch.zeros((2, 3, dim), dtype=torch.float16, device=dev)
    q[1, :, 0] = 1.0
    got = blockedAttention.pagedAttention(q, k, v, table, lens, 1.0)
    for r in range(2):
        n = lens[r].item()
        mean = ((width - 1) * page + 3 * (n - (width - 1) * page - 200) + last[r].double().sum(0)) / n
        assert ((got[0, r].double() - mean).abs() <= 2.0 ** -11 * mean.abs() + 2.0 ** -20).all()
        assert torch.equal(got[1, r], last[r, -1])
    assert (got[:, 2] == 1).all()
    # the window's part alone: as the same tokens at the beginning of a request
    q = (torch.randn((2, 3, dim), generator=g) * 2).half().to(dev)
    k[1:, 0, -300:-3] = (torch.randn((2, 297, dim), generator=g)).half().to(dev)
    got = blockedAttention.pagedAttention(q, k, v, table, lens, 0.5, 100)
    for r in range(2):
        n = page - 3 * r
        p = torch.softmax(q[:, r].double() @ k[r + 1, 0, n - 100:n].double().t() * 0.5, -1)
        want = p @ v[r + 1, 0, n - 100:n].double()
        assert ((got[:, r].double() - want).abs() <= 2.0 ** -9 * (p @ v[r + 1, 0, n - 100:n].double().abs()) + 2.0 ** -20).all()
