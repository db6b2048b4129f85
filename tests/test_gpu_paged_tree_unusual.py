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


@pytest.mark.parametrize("dtype,fp8", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float16, False), (torch.float16, True)])
@pytest.mark.parametrize("dim,nodes", [(64, 12), (64, 40), (128, 40), (256, 40), (100, 40), (128, 3)])
def test_probabilities_have_more_than_16_bits(dev, roomy, monkeypatch, dtype, fp8, dim, nodes):  # noqa: F811
    """The result's own rounding is the only one to 16 bits, whichever kernel a batch takes.

    Bound: as in test_gpu_paged_tree_attention.py, but a probability p is off by 2^-16 p at most (two terms, the first cut off: bf16 2^-7 x 2^-9, fp16 less), in
    fp16 by half a step of 2^-24 besides, or a whole one where the second term is made that, lifted by 2^8 against the largest: 2^-31 of it a token.  bf16 over e4m3: one fp16 term, off
    by 2^-11 p, and so is the sum of them that it is divided by: 2^-10 together (the kernel for few rows: two terms).
    """
    b = Drafts([300, 77, 0], [nodes, nodes, nodes], 2, 4, dim, 16, dtype, fp8, mask="tree", seed=dim)
    import test_gpu_paged_tree_attention as base
    u = base.U[dtype]
    monkeypatch.setitem(base.U, dtype, 0.0)
    ref, rest = b.expect(dim ** -0.5)
    monkeypatch.setitem(base.U, dtype, 1.0)
    size = b.expect(dim ** -0.5)[1] - rest - ref.abs()
    most = torch.nan_to_num(b.v.float()).abs().max().item() * (max(b.scales[1]).item() if fp8 else 1.0)
    term = 2.0 ** -10 if fp8 and dtype == torch.bfloat16 else 2.0 ** -16
    bound = u * ref.abs() + rest + term * size + 400 * 2.0 ** -31 * most
    got = b.run(dev, dim ** -0.5).double().cpu()
    assert ((got - ref).abs() <= bound).all(), (((got - ref).abs() - bound).max().item(), ((got - ref).abs() > bound).double().mean().item())


@pytest.mark.parametrize("lens,nodes,heads,group,dim,fp8", [
    (12000, 3, 1, 4, 128, False), (12000, 7, 2, 4, 64, True), (1500, 4, 8, 4, 128, False), (1500, 7, 8, 4, 64, False),      # few rows: joined by a second kernel, within the kernel
    (12000, 40, 1, 4, 128, False), (12000, 40, 1, 4, 128, True), (9000, 12, 1, 4, 64, False), (9000, 40, 1, 4, 256, False)])
@pytest.mark.parametrize("far", [False, True])
def test_units_of_several_workgroups(dev, lens, nodes, heads, group, dim, fp8, far):
    """Infinities and NaN among the drafted values of a long request; far: its first token outweighs the part that they are in by more than fp32 holds."""
    b = Drafts([lens], [nodes], heads, group, dim, 16, torch.float16, fp8, mask="any", seed=nodes)
    if far:
        b.q.zero_()
        b.q[..., 0] = 16.0
        k = torch.zeros((heads, 1, dim), dtype=torch.float16)
        k[..., 0] = 40.0
        if fp8:
            b.scales[0].fill_(1.0)
            b.k = (b.k.float() / 128).to(FP8)
        b.put(b.k, 0, 0, k.to(FP8) if fp8 else k)
    scale = 1.0 if far else 0.125
    ref, bound = b.expect(scale)
    put_value(b, 0, 1, torch.nan, 3)
    if not fp8:
        put_value(b, 0, 2, torch.inf, 5)
    got = b.run(dev, scale).double().cpu()
    usual = torch.ones(dim, dtype=torch.bool)
    usual[[3, 5]] = False
    for i in range(nodes):
        x, y = bool(b.sees[0][i, 1]), bool(b.sees[0][i, 2]) and not fp8
        near = (got[:, i] - ref[:, i]).abs() <= bound[:, i]
        if not x and not y:
            assert near.all(), i
            continue
        if far:                                               # (else the zeros that were put there change the other dimensions)
            assert near[:, usual].all(), i
        assert (got[:, i, 3].isnan() if x else got[:, i, 3].isfinite()).all(), (i, got[:, i, 3])
        assert (got[:, i, 5] == torch.inf if y else got[:, i, 5].isfinite()).all(), (i, got[:, i, 5])
    assert b.sees[0][:, 1].any() and b.sees[0][:, 2].any()


@pytest.mark.parametrize("nodes,room", [(6, 0), (30, 4096)])
@pytest.mark.parametrize("base,window", [(1000, 0), (1000, 40), (1000, 64), (1024, 33), (1000, 300), (1000, 1010), (3, 1)])
def test_places_of_values_that_are_not_finite(dev, monkeypatch, nodes, room, base, window):
    """A NaN at each place in turn that not all rows see, and its neighbours: where windows begin, in the draft, both, or where they meet."""
    monkeypatch.setattr(Drafts, "room", room)
    b = Drafts([base], [nodes], 1, 4, 64, 16, torch.float16, mask="tree", seed=base + window)
    ref, bound = b.expect(0.125, window)
    sees = b.seen(0, window)                                  # [nodes, tokens]
    some = (sees.any(0) != sees.all(0)).nonzero()[:, 0].tolist()
    for t in sorted({x for t in some for x in (t - 1, t, t + 1) if 0 <= x < base + nodes})[::3]:
        at = (int(b.table[0, t // 16]), slice(None), t % 16)
        old = b.v[at].clone()
        b.v[at] = torch.nan
        b.__dict__.pop("there", None)
        got = b.run(dev, 0.125, window).double().cpu()
        b.v[at] = old
        assert got[:, sees[:, t]].isnan().all(), t
        assert ((got - ref).abs() <= bound)[:, ~sees[:, t]].all(), t


@pytest.mark.parametrize("nodes", [3, 8, 40])
@pytest.mark.parametrize("dim,fp8", [(64, False), (128, True), (100, False), (7, False)])
def test_rows_that_see_nothing_whatever_the_scale(dev, roomy, nodes, dim, fp8):  # noqa: F811
    """Zeros, beside rows of the same unit that see tokens and are NaN where the scale is."""
    b = Drafts([0], [nodes], 2, 4, dim, 16, torch.bfloat16, fp8, mask="any", seed=3, pad=2)
    b.sees[0][1] = False
    b.mask[1] = 0
    b.sees[0][2, 0] = True
    b.mask[2, 0] |= 1
    none = ~b.sees[0].any(1)
    for scale in (float("nan"), float("inf"), -float("inf")):
        got = b.run(dev, scale)
        assert (got[:, :nodes][:, none] == 0).all() and (got[:, nodes:] == 0).all()
        if scale != scale:
            assert got[:, :nodes][:, ~none].isnan().all()


@pytest.mark.parametrize("nodes", [3, 8, 40])
@pytest.mark.parametrize("scale", [2.0 ** -125, -2.0 ** -127, 2.0 ** -131, 2.0 ** -149, 0.0])
def test_large_scores_of_a_tiny_scale(dev, roomy, nodes, scale):  # noqa: F811
    """Scores of up to 2^124 before they are scaled.  Where the scale is a number of few bits, times log2(e) it is off by 2^-150, half the smallest one: 2^-26 of a score's exponent."""
    b = Drafts([70, 0], [nodes, nodes], 2, 4, 64, 16, torch.bfloat16, mask="tree", seed=nodes)
    b.q *= 2.0 ** 58
    b.k *= 2.0 ** 58
    b.check(dev, scale)


@pytest.mark.parametrize("base,nodes", [(0, 3), (0, 9), (0, 40), (70, 3), (70, 40), (6000, 3), (6000, 40)])
@pytest.mark.parametrize("mask", ["any", "chain"])
def test_scores_that_are_all_minus_infinity(dev, roomy, base, nodes, mask):  # noqa: F811
    """No probability is above 0: zeros, as for a row that sees nothing; also where a request is split between workgroups."""
    b = Drafts([base, 50], [nodes, nodes], 2, 4, 64, 16, torch.float16, mask=mask, seed=nodes)
    ref, bound = b.expect(1.0)
    b.q[:, :nodes] = 0.0
    b.q[:, :nodes, 0] = 1.0
    x = torch.zeros((2, base + nodes, 64), dtype=torch.float16)
    x[..., 0] = -torch.inf
    b.put(b.k, 0, 0, x)
    got = b.run(dev, 1.0).double().cpu()
    assert (got[:, :nodes] == 0).all()
    assert ((got - ref).abs() <= bound)[:, nodes:].all()
