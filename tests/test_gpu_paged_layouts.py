"""Operands of the paged cache's operators in unusual layouts: the same values in the usual one give the same bits."""
import pytest
import torch

import blockedAttention
from test_gpu_paged_attention import Batch

pytestmark = pytest.mark.gpu

# queries of four heads, three requests, dimension 16 as views of 400 numbers
QUERIES = {
    "rows one element apart": lambda x: x[:4 * 18].view(4, 18).unfold(-1, 16, 1),
    "rows and heads one element apart": lambda x: x.as_strided((4, 3, 16), (1, 1, 1)),
    "heads one element apart, rows inside": lambda x: x.as_strided((4, 3, 16), (1, 40, 1)),
    "heads by dimensions one element apart": lambda x: x.as_strided((4, 48), (1, 1)),
    "one row for all": lambda x: x[:16].expand(4, 3, 16),
    "one head for all": lambda x: x[:48].expand(4, 48),
    "requests outside": lambda x: x[:4 * 48].view(3, 4, 16).transpose(0, 1),
    "padded": lambda x: x[:4 * 3 * 20].view(4, 3, 20)[..., 1:17],
}


@pytest.mark.parametrize("name", QUERIES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_queries(dev, name, dtype):
    b = Batch([40, 0, 700], 2, 2, 16, 16, dtype, seed=3)
    q = QUERIES[name]((torch.randn(400, generator=torch.Generator().manual_seed(1)) * 2).to(dtype).to(dev))
    rest = (b.k.to(dev), b.v.to(dev), b.table.to(dev), torch.tensor(b.lens).to(dev), 0.25)
    want = blockedAttention.pagedAttention(q.contiguous(), *rest)
    got = blockedAttention.pagedAttention(q, *rest)
    assert got.shape == q.shape and got.dtype == dtype
    assert torch.equal(got, want)


def test_a_table_row_that_all_requests_share(dev):
    """One row of pages, expanded over the requests: a prefix that all of them have, seen to different lengths."""
    b = Batch([300], 2, 4, 64, 16, torch.float16, seed=5)
    q = torch.randn((8, 5, 64), generator=torch.Generator().manual_seed(2)).half().to(dev)
    lens = torch.tensor([300, 0, 17, 128, 1], device=dev)
    k, v, row = b.k.to(dev), b.v.to(dev), b.table.to(dev)
    got = blockedAttention.pagedAttention(q, k, v, row.expand(5, -1), lens, 0.125)
    assert torch.equal(got, blockedAttention.pagedAttention(q, k, v, row.repeat(5, 1), lens, 0.125))
    with pytest.raises(RuntimeError):                                     # where rows are written they have to be apart
        blockedAttention.pagedResize(row.expand(5, -1), torch.arange(9, dtype=torch.int32, device=dev), torch.tensor([9, 0], device=dev),
                                     lens, lens, 16, 0)


@pytest.mark.parametrize("fp8", [False, True])
def test_strides_of_dimensions_of_one(dev, fp8):
    """Pages of one token, one page, one head: the stride of a dimension of one means nothing, however large."""
    for lens, heads, page in (([5, 9], 2, 1), ([7], 2, 16), ([40, 3], 1, 16)):
        b = Batch(lens, heads, 2, 32, page, torch.float16, fp8, seed=page, extra=0)
        k, v, q, table, lens = b.k.to(dev), b.v.to(dev), b.q.to(dev), b.table.to(dev), torch.tensor(lens).to(dev)
        scales = [None if s is None else s.to(dev) for s in b.scales]
        want = blockedAttention.pagedAttention(q, k, v, table, lens, 0.25, 0, *scales)
        far = [c.as_strided(c.shape, [(1 << 45) + 1 if n == 1 else s for n, s in zip(c.shape, c.stride())]) for c in (k, v)]
        assert torch.equal(blockedAttention.pagedAttention(q, *far, table, lens, 0.25, 0, *scales), want)
        x = torch.randn((heads, 1, 32), device=dev).half()
        place = torch.tensor([page * k.size(0) - 1], device=dev)
        blockedAttention.pagedAppend(x, 2 * x, k, v, place, *scales)
        want = [c.clone().view(torch.uint8) for c in (k, v)]
        for c in (k, v):
            c.view(torch.uint8).zero_()
        blockedAttention.pagedAppend(x, 2 * x, *far, place, *scales)
        for c, w in zip((k, v), want):
            last = (k.size(0) - 1, slice(None), page - 1)
            assert torch.equal(c.view(torch.uint8)[last], w[last]) and c.view(torch.uint8)[last].any()


def test_scales_that_want_gradients_are_refused(dev):
    """There is no backward pass: a scale that is trained would silently get no gradient."""
    b = Batch([20], 2, 2, 64, 16, torch.float16, True)
    q, k, v, table, lens = b.q.to(dev), b.k.to(dev), b.v.to(dev), b.table.to(dev), torch.tensor(b.lens, device=dev)
    plain, trained = b.scales[0].to(dev), b.scales[0].to(dev).requires_grad_()
    x, slots = q[:2], torch.zeros(1, dtype=torch.int64, device=dev)
    for scales in ((plain, trained), (trained, plain)):
        with pytest.raises(RuntimeError, match="no backward pass"):
            blockedAttention.pagedAttention(q, k, v, table, lens, 0.1, 0, *scales)
        with pytest.raises(RuntimeError, match="no backward pass"):
            blockedAttention.pagedAppend(x, x, k, v, slots, *scales)
        with torch.no_grad():
            blockedAttention.pagedAppend(x, x, k, v, slots, *scales)
            blockedAttention.pagedAttention(q, k, v, table, lens, 0.1, 0, *scales)
