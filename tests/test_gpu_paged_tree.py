"""pagedTree against sets built node by node."""
import pytest
import torch

import blockedAttention

pytestmark = pytest.mark.gpu


def plain(parents, accum, nodes, tokens):
    words = -(-nodes // 64)
    mask, depth = [[0] * words for _ in range(tokens)], [-1] * tokens
    for a, b in zip(accum, accum[1:]):
        sees = {}
        for i in range(min(b, tokens) - a):
            p = parents[a + i]
            if i >= nodes or not -1 <= p < i or (p >= 0 and p not in sees):
                continue
            sees[i] = (sees[p] if p >= 0 else 0) | 1 << i
            depth[a + i] = bin(sees[i]).count("1") - 1
            for w in range(words):
                x = sees[i] >> 64 * w & (1 << 64) - 1
                mask[a + i][w] = x - (1 << 64) if x >> 63 else x
    return torch.tensor(mask, dtype=torch.int64).reshape(tokens, words), torch.tensor(depth, dtype=torch.int64)


def check(dev, parents, sizes, nodes, pad=0, front=0):
    accum = [front]
    for n in sizes:
        accum.append(accum[-1] + n)
    tokens = accum[-1] + pad
    parents = [7] * front + parents + [3] * pad
    got = blockedAttention.pagedTree(torch.tensor(parents, device=dev, dtype=torch.int64), torch.tensor(accum, device=dev), nodes)
    want = plain(parents, accum, nodes, tokens)
    for g, w in zip(got, want):
        assert g.dtype == torch.int64 and torch.equal(g.cpu(), w)


def shaped(shape, n, g):
    if shape == "chain":
        return list(range(-1, n - 1))
    if shape == "star":
        return [-1] * n
    if shape == "comb":                                       # a long chain with a leaf at every node
        return [-1 if i < 2 else i - 2 + i % 2 * -1 for i in range(n)]
    return [int(torch.randint(-1, i, (1,), generator=g)) if i else -1 for i in range(n)]


@pytest.mark.parametrize("shape", ["chain", "star", "comb", "random"])
@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 128, 129, 300, 1000, 1024])
def test_shapes(dev, shape, n):
    check(dev, shaped(shape, n, torch.Generator().manual_seed(n)), [n], n)


@pytest.mark.parametrize("sizes,nodes", [([0, 5, 0, 70, 1, 0], 70), ([3, 3], 64), ([130, 1, 64, 200], 200), ([0, 0], 1), ([40] * 300, 40)])
@pytest.mark.parametrize("pad,front", [(0, 0), (13, 0), (2100, 5)])
def test_ragged_batches(dev, sizes, nodes, pad, front):
    g = torch.Generator().manual_seed(5)
    check(dev, sum((shaped("random", n, g) for n in sizes), []), sizes, nodes, pad, front)


def test_no_requests_and_no_tokens(dev):
    check(dev, [], [], 4, pad=9)
    check(dev, [], [0, 0, 0], 4)
    check(dev, [], [], 4)


def test_nodes_without_a_parent_before_them(dev):
    """A parent that is no earlier node, at every place of a block, and what goes on from such nodes."""
    g = torch.Generator().manual_seed(3)
    for n, bad in ((40, [7]), (200, [0, 63, 64, 130]), (200, [5]), (1024, [511, 900])):
        for value in (-2, None, 10 ** 12, -(1 << 62)):
            parents = shaped("random", n, g)
            for i in bad:
                parents[i] = i if value is None else value
            check(dev, parents, [n], n)


def test_more_nodes_than_said(dev):
    check(dev, shaped("chain", 100, None) * 2, [100, 100], 70)
    check(dev, shaped("star", 100, None), [100], 64)


def test_rows_beyond_the_tokens_are_not_written(dev):
    """Sums that end behind the arrays."""
    back = torch.full((40,), 77, dtype=torch.int64, device=dev)
    parents = torch.arange(-1, 9, device=dev)
    from blockedattention_amd import capi
    mask, depth = back[:10].view(10, 1), back[20:30]
    capi.paged_tree(parents, torch.tensor([0, 6, 25], device=dev), 64, mask, depth)
    assert (back[10:20] == 77).all() and (back[30:] == 77).all()
    assert back[20:30].tolist() == [0, 1, 2, 3, 4, 5, -1, -1, -1, -1]         # (parents 5.. come after nodes 0..)


def test_on_another_stream_and_in_a_graph(dev):
    g = torch.Generator().manual_seed(1)
    sizes = [50, 90, 3]
    accum = torch.tensor([0, 50, 140, 143], device=dev)
    trees = [sum((shaped("random", n, g) for n in sizes), []) for _ in range(3)]
    parents = torch.tensor(trees[0], device=dev)
    blockedAttention.pagedTree(parents, accum, 90)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = blockedAttention.pagedTree(parents, accum, 90)
    for t in trees:
        parents.copy_(torch.tensor(t))
        graph.replay()
        torch.cuda.synchronize()
        want = plain(t, accum.tolist(), 90, 143)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(out, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = blockedAttention.pagedTree(parents, accum, 90)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, out))
