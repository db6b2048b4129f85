"""pagedTreeAttention where values that are not finite, infinite scores and unusual scales meet workgroups of several units and units of several workgroups.

Rows that see nothing unusual are within the bound of test_gpu_paged_tree_attention.py.
"""
import pytest
import torch

from test_gpu_paged_tree_attention import FP8, Drafts, roomy  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def put_value(b, r, node, value, dims=slice(None)):
    """Value of a node: `value` in some of its dimensions, zeros in the others."""
    x = torch.zeros((b.heads, 1, b.dim), dtype=b.dtype)
    x[..., dims] = value
    b.put(b.v, r, b.base[r] + node, x.to(FP8) if b.fp8 else x)


@pytest.mark.parametrize("dim,fp8,nodes", [(64, False, 6), (64, False, 14), (128, False, 6), (128, True, 14), (256, False, 4), (64, False, 26), (128, True, 40), (256, False, 40)])
def test_workgroups_of_several_units(dev, roomy, dim, fp8, nodes):  # noqa: F811
    """More units than workgroups, every third with a NaN among its drafted values: a unit's end and the next one's beginning do not mix."""
    g = torch.Generator().manual_seed(nodes)
    n = torch.randint(2, nodes, (900,), generator=g).tolist()
    b = Drafts(torch.randint(0, 60, (900,), generator=g).tolist(), n, 2, 4, dim, 16, torch.float16, fp8, mask="any", seed=dim)
    ref, bound = b.expect(0.125)
    odd = {r: r % n[r] for r in range(0, 900, 3)}
    for r, node in odd.items():
        put_value(b, r, node, torch.nan)
    got = b.run(dev, 0.125).double().cpu()
    sees = torch.zeros(b.tokens, dtype=torch.bool)
    for r, node in odd.items():
        sees[b.accum[r]:b.accum[r + 1]] = b.sees[r][:, node]
    assert sees.any() and got[:, sees].isnan().all()
    assert ((got - ref).abs() <= bound)[:, ~sees].all()
