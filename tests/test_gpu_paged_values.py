"""pagedAttention: what infinite values, and probabilities that are no 16-bit number, do to the result."""
import pytest
import torch

from test_gpu_paged_attention import Batch

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
