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
