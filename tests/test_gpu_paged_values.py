"""pagedAttention: what infinite values, and probabilities that are no 16-bit number, do to the result."""
import pytest
import torch

from test_gpu_paged_attention import FP8, U, Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,group,lens", [(64, 2, [1, 5, 64, 333]), (100, 17, [3, 40]), (128, 4, [2, 100, 5000]), (256, 1, [1, 70])])
@pytest.mark.parametrize("alike", [False, True])
def test_an_infinite_value_that_counts_makes_its_column_infinite(dev, dtype, dim, group, lens, alike):
    """A token's probability is above zero, so what it has infinite is infinite in the result, with its sign; two signs give NaN.

    `alike`: all tokens of a request have the same probability, which is a 16-bit number where there are 1, 2, 4, ...
    """
    b = Batch(lens, 2, group, dim, 16, dtype, seed=dim, spread=0.0 if alike else 1.0)
    for r, n in enumerate(lens):
        for t, d, sign in ((0, 0, 1), (n - 1, 1, -1), (n // 2, dim - 1, 1), (0, 2, 1), (n // 3, 3, -1), (n - 1, 2, -1)):
            b.v[int(b.table[r, t // 16]), :, t % 16, d] = sign * float("inf")
    scale = dim ** -0.5
    got = b.run(dev, scale).double().cpu()
    ref, bound = b.expect(scale)
    finite = torch.isfinite(ref)
    assert not finite[..., 0].any() and finite[..., 4].all()
    # (NaN only where both signs meet)
    assert torch.equal(torch.nan_to_num(got[~finite], nan=0.5), torch.nan_to_num(ref[~finite], nan=0.5))
    assert ((got - ref).abs() <= bound)[finite].all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_probability_is_kept_to_more_than_16_bits(dev, dtype, fp8, dim):
    """128 tokens whose signed values nearly cancel: the rounding of the result is small, that of the probabilities is not.

    Bound, times P |V|: what two 16-bit terms lose of a probability, 2^-16 (bf16, 8 bits a term) or 2^-21 (fp16, 11 bits; those
    here are far above its smallest number); 2 (2 + 8) 2^-24 max |scale| sum |q k| for scores of two non-zero products in fp32;
    2^-20 for the exponentials; 80 additions of fp32 (a tile's 64 products, four wavefronts).  And the result's own rounding.
    """
    heads, n = 4, 128
    b = Batch([n], heads, 1, dim, 16, dtype, fp8, seed=dim)
    g = torch.Generator().manual_seed(dim + 1)
    b.q[:] = 0
    b.q[:, 0, :2] = torch.randn((heads, 2), generator=g).to(dtype)
    k = torch.randint(-16, 17, (heads, n, dim), generator=g) / 8.0
    q = b.q[:, 0].double()
    p = torch.softmax(torch.matmul(k.double(), q[:, :, None])[..., 0], -1)                  # [heads, tokens]
    v = torch.randint(8, 16, (heads, n, dim), generator=g) / 8.0
    order, total = p.argsort(-1, descending=True), torch.zeros((heads, dim), dtype=torch.float64)
    for i in range(n):                                                                      # signs that keep the sum near 0
        at = (torch.arange(heads), order[:, i])
        v[at] *= torch.where(total > 0, -1.0, 1.0)
        total += p[at][:, None] * v[at]
    for c, x in ((b.k, k), (b.v, v)):
        raw, mine = (c.view(torch.uint8), x.to(FP8).view(torch.uint8)) if fp8 else (c, x.to(dtype))
        for i in range(n // 16):
            raw[int(b.table[0, i])] = mine[:, 16 * i:16 * i + 16]
    if fp8:
        b.scales = [torch.ones(heads), torch.ones(heads)]
    got = b.run(dev, 1.0).double().cpu()[:, 0]
    e = 10 * 2.0 ** -24 * (k.double().abs() * q.abs()[:, None]).sum(-1).amax(-1)
    terms = 2.0 ** -16 if dtype == torch.bfloat16 else 2.0 ** -21
    ref, size = (torch.matmul(p[:, None], x.double())[:, 0] for x in (v, v.abs()))
    bound = U[dtype] * ref.abs() + (terms + 2 * e[:, None] + 2.0 ** -20 + 80 * 2.0 ** -24) * size + 2.0 ** -24
    one = torch.matmul(p.to(dtype).double()[:, None], v.double())[:, 0]                     # with one 16-bit term each
    assert ((one - ref).abs() > 2 * bound).any()
    assert ((got - ref).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("size", [2.0 ** 12, 3.0 * 2 ** 12, 2.0 ** 14, 3.0 * 2 ** 14, 60000.0])
def test_scores_of_many_millions_find_their_token(dev, dtype, fp8, size):
    """One key is far closer to the query than all others: the result is its value, whatever the scores' last digits are worth."""
    b = Batch([1, 100, 700], 2, 2, 64, 16, dtype, fp8, seed=21)
    b.q[:] = 0
    b.q[..., :16] = size
    b.scales = [torch.ones(2), torch.ones(2)] if fp8 else [None, None]
    top = torch.tensor(448.0 if fp8 else size).to(b.k.dtype)
    want = torch.zeros(b.q.shape, dtype=torch.float64)
    for r, n in enumerate(b.lens):
        for t in range(n):
            at = (int(b.table[r, t // 16]), slice(None), t % 16)
            row = torch.zeros((2, 64)).to(b.k.dtype)
            for c in range(16 if t == n // 3 else t % 3):                 # 16 times the size, or not even a fifth of that
                row.view(torch.uint8 if fp8 else torch.int16)[:, c] = top.view(torch.uint8 if fp8 else torch.int16)
            b.k.view(row.view(torch.uint8).dtype if fp8 else torch.int16)[at] = row.view(torch.uint8 if fp8 else torch.int16)
        v = b.tokens(b.v, b.scales[1], r, 0, n)
        want[:, r] = v[:, n // 3].repeat_interleave(2, 0)
    for scale, other in ((1.0, None), (0.125, None), (-1.0, 0)):
        if other is None:
            got = b.run(dev, scale).double().cpu()
            assert torch.equal(got, want.to(dtype).double()), scale
        else:
            assert torch.isfinite(b.run(dev, scale)).all()
