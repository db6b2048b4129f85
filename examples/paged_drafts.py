"""Drafted and branching answers through one attention layer with a paged key-value cache.

    python examples/paged_drafts.py [--cache fp8]

Every step each row gets new tokens: an empty one a prompt, the others a tree of guesses at how they go on.

    pagedResize         gives the new tokens their places
    pagedTree           says what each of them sees, and how deep it lies
    pagedAppend         writes keys and values of all to their places
    pagedTreeAttention  attends from each new token to all that it sees
    pagedKeep           moves the accepted branch of each tree to its front; pagedResize then gives the other pages back
    pagedFork           lets rows go on from other rows, as beams and samples do, and ends rows; their pages are shared
    pagedCopy           copies the last pages, which are written next

The host draws the trees and what is accepted; the GPU keeps pages and places, and nothing waits for it until the end, when the verdict of all
steps is read.  The weights are random; every result is compared with the same over dense copies in fp32.
"""
import argparse
import os
import random
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import blockedAttention  # noqa: E402

ROWS, HEADS, GROUP, DIM, PAGE, LONGEST, NODES = 12, 2, 4, 64, 16, 320, 48      # rows of the table; key heads; query heads of each
HIDDEN = 256
FP8 = torch.float8_e4m3fn


class Layer:
    def __init__(self, dev, cache_dtype, dtype=torch.bfloat16):
        weight = lambda n: (torch.randn((HIDDEN, n * DIM), device=dev) * HIDDEN ** -0.5).to(dtype)  # noqa: E731
        self.wq, self.wk, self.wv = weight(HEADS * GROUP), weight(HEADS), weight(HEADS)
        self.pages = ROWS * LONGEST // PAGE
        self.k, self.v = (torch.zeros((self.pages, HEADS, PAGE, DIM), device=dev).to(cache_dtype) for _ in range(2))
        self.scales = [torch.full((HEADS,), 4.0 / 448, device=dev) for _ in range(2)] if cache_dtype == FP8 else [None, None]
        self.places = (torch.randn((LONGEST, HIDDEN), device=dev) * 0.5).to(dtype)       # added by a token's position

    def project(self, x, w):
        return (x @ w).view(len(x), -1, DIM).transpose(0, 1)          # [heads, tokens, dim], rows of the product

    def stored(self, t, which):
        """What the cache has of [heads, tokens, dim], in fp32."""
        if self.scales[which] is None:
            return t.float()
        scale = self.scales[which][:, None, None]
        return (t.float() / scale).clamp(-448, 448).to(FP8).float() * scale


def branch(parents, node):
    """The nodes from a tree's root to one of its nodes."""
    path = []
    while node >= 0:
        path.append(node)
        node = parents[node]
    return path[::-1]


def main(cache="bf16", steps=40, seed=0):
    dev = torch.device("cuda")
    torch.manual_seed(seed)
    rng = random.Random(seed)
    layer = Layer(dev, FP8 if cache == "fp8" else torch.bfloat16)
    table = torch.zeros((ROWS, LONGEST // PAGE), dtype=torch.int32, device=dev)
    free = torch.arange(layer.pages, dtype=torch.int32, device=dev)
    state = torch.tensor([layer.pages, 0], device=dev)
    shares = torch.zeros(layer.pages, dtype=torch.int32, device=dev)
    lens = torch.zeros(ROWS, dtype=torch.int64, device=dev)
    have = [0] * ROWS                                                 # the host's copy of the lengths
    nothing = torch.zeros((HEADS, 0, DIM), device=dev)
    dense = [(nothing, nothing)] * ROWS                               # for the comparison: keys and values
    worst, answered, forked = 0.0, 0, 0
    for step in range(steps):
        # prompts, which are chains, and trees; every fourth step all guesses are chains too, which need no mask
        chains = step % 4 == 3
        parents = []
        for r in range(ROWS):
            n = rng.randint(1, NODES) if have[r] == 0 else rng.randint(0, 12)
            parents.append([i - 1 if have[r] == 0 or chains else rng.randint(-1, i - 1) for i in range(n)])
        counts = [len(p) for p in parents]
        tokens, at = sum(counts), [sum(counts[:r]) for r in range(ROWS)]
        new = torch.tensor([h + n for h, n in zip(have, counts)], device=dev)
        slots, accum, grown, state = blockedAttention.pagedResize(table, free, state, lens, new, PAGE, tokens)

        mask, depth = blockedAttention.pagedTree(torch.tensor([p for row in parents for p in row], device=dev), accum, NODES)
        row = torch.tensor([r for r in range(ROWS) for _ in parents[r]], device=dev)
        x = torch.randn((tokens, HIDDEN), device=dev).bfloat16() + layer.places[lens[row] + depth]
        q, k, v = (layer.project(x, w) for w in (layer.wq, layer.wk, layer.wv))
        blockedAttention.pagedAppend(k, v, layer.k, layer.v, slots, *layer.scales)
        out = blockedAttention.pagedTreeAttention(q, layer.k, layer.v, table, grown, accum, None if chains else mask, scale=DIM ** -0.5,
                                                  kScale=layer.scales[0], vScale=layer.scales[1])

        # one branch of each tree is accepted, all of a prompt
        paths = []
        for r, p in enumerate(parents):
            path = branch(p, rng.randrange(len(p))) if p else []
            if have[r]:
                path = path[:rng.randint(0, len(path))]
            else:
                path = list(range(len(p)))
            mine = [layer.stored(t[:, at[r]:at[r] + counts[r]], i) for i, t in enumerate((k, v))]
            for i in range(counts[r]):
                seen = branch(p, i)
                kr, vr = (torch.cat([d, m[:, seen]], 1) for d, m in zip(dense[r], mine))
                w = torch.softmax(q[:, at[r] + i].float().view(HEADS, GROUP, DIM) @ kr.transpose(1, 2) * DIM ** -0.5, -1)
                worst = max(worst, (w @ vr - out[:, at[r] + i].float().view(HEADS, GROUP, DIM)).abs().max().item())
                answered += 1
            dense[r] = tuple(torch.cat([d, m[:, path]], 1) for d, m in zip(dense[r], mine))
            have[r] += len(path)
            paths.append(path)
        deepest = max(map(len, paths))
        path = torch.tensor([p + [-1] * (deepest - len(p)) for p in paths], dtype=torch.int64, device=dev).reshape(ROWS, deepest)
        path = torch.where(state[1] == 0, path, -1)                       # (a step that was refused gave its tokens no places)
        kept = blockedAttention.pagedKeep(layer.k, layer.v, table, lens, path)
        _, _, lens, state = blockedAttention.pagedResize(table, free, state, grown, kept, PAGE, 0)

        # long rows end, some others too; empty places go on from rows that are there
        origin = [-1 if have[r] > LONGEST - NODES or rng.random() < 0.1 else r for r in range(ROWS)]
        there = [r for r in range(ROWS) if origin[r] == r and have[r]]
        for r in range(ROWS):
            if (origin[r] < 0 or have[r] == 0) and there and rng.random() < 0.6:
                origin[r] = rng.choice(there)
                forked += 1
        table, lens, state, shares, source, target = blockedAttention.pagedFork(table, free, state, shares, lens, torch.tensor(origin, device=dev), PAGE)
        blockedAttention.pagedCopy(layer.k, layer.v, source, target)
        have, dense = [have[o] if o >= 0 else 0 for o in origin], [dense[o] if o >= 0 else (nothing, nothing) for o in origin]
    assert state[1].item() == 0, f"a step was refused: verdict {state[1].item()}"
    assert lens.tolist() == have
    # all rows end: every page is free again, and nobody's
    table, lens, state, shares, _, _ = blockedAttention.pagedFork(table, free, state, shares, lens, torch.full((ROWS,), -1, device=dev), PAGE)
    assert state.tolist() == [layer.pages, 0] and sorted(free.tolist()) == list(range(layer.pages)) and not shares.any() and not lens.any()
    return worst, answered, forked


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--cache", choices=["bf16", "fp8"], default="bf16")
    parser.add_argument("--steps", type=int, default=40)
    args = parser.parse_args()
    error, count, rows = main(args.cache, args.steps)
    print(f"{count} tokens answered, {rows} rows gone on from others, largest difference from dense attention in fp32: {error:.3g}")
