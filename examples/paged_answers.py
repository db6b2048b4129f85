"""Answers to a changing batch of requests through one attention layer with a paged key-value cache.

    python examples/paged_answers.py [--cache fp8]

Every step some requests arrive with a prompt, some end, the others go on by one token:

    pagedResize          gives the prompts and the new tokens their places, and the ended requests' pages to others
    blockFusedAttention  attends within the prompts (segments of different lengths back to back), from every token to all of
                         its prompt: it has no causal mask, so this is a prefix that is read in both directions
    pagedAppend          writes keys and values of both to their places
    pagedAttention       attends from each request's new token to all that it has

The host makes the lengths; the GPU keeps pages and places, and nothing waits for it until the end, when the verdict of
all steps is read.  The weights are random; every result of either attention is compared with the same over dense copies in fp32.
"""
import argparse
import os
import random
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import blockedAttention  # noqa: E402

SLOTS, HEADS, GROUP, DIM, PAGE, LONGEST = 12, 2, 4, 64, 16, 256       # requests at a time; key heads; query heads of each
HIDDEN = 256


class Layer:
    def __init__(self, dev, cache_dtype, dtype=torch.bfloat16):
        weight = lambda n: (torch.randn((HIDDEN, n * DIM), device=dev) * HIDDEN ** -0.5).to(dtype)  # noqa: E731
        self.wq, self.wk, self.wv = weight(HEADS * GROUP), weight(HEADS), weight(HEADS)
        pages = SLOTS * LONGEST // PAGE * 3 // 4                      # fewer than all requests at full length would need
        self.k, self.v = (torch.zeros((pages, HEADS, PAGE, DIM), device=dev).to(cache_dtype) for _ in range(2))
        self.scales = [torch.full((HEADS,), 4.0 / 448, device=dev) for _ in range(2)] if cache_dtype == torch.float8_e4m3fn else [None, None]

    def project(self, x, w):
        return (x @ w).view(len(x), -1, DIM).transpose(0, 1)          # [heads, tokens, dim], rows of the product


def main(cache="bf16", steps=40, seed=0):
    dev = torch.device("cuda")
    torch.manual_seed(seed)
    rng = random.Random(seed)
    layer = Layer(dev, torch.float8_e4m3fn if cache == "fp8" else torch.bfloat16)
    pages = layer.k.shape[0]
    table = torch.zeros((SLOTS, LONGEST // PAGE), dtype=torch.int32, device=dev)
    free = torch.arange(pages, dtype=torch.int32, device=dev)
    state = torch.tensor([pages, 0], device=dev)
    lens = torch.zeros(SLOTS, dtype=torch.int64, device=dev)
    have = [0] * SLOTS                                                # the host's copy of the lengths
    dense = [[None, None] for _ in range(SLOTS)]                      # for the comparison: keys and values, [heads, tokens, dim]
    worst, answered = 0.0, 0
    for step in range(steps):
        # which requests end, arrive with a prompt or go on: each is a change of length
        prompts, new = [], list(have)
        used = sum(-(-n // PAGE) + 1 for n in have)
        for r in range(SLOTS):
            if have[r] == 0:
                n = rng.randint(1, LONGEST // 2)
                if rng.random() < 0.5 and used + n // PAGE + 2 < pages:
                    new[r], used = n, used + n // PAGE + 2
                    prompts.append(r)
            elif have[r] >= LONGEST or rng.random() < 0.05:
                new[r] = 0
            else:
                new[r] += 1
        grown = [max(n - o, 0) for o, n in zip(have, new)]
        tokens = sum(grown)
        slots, _, lens, state = blockedAttention.pagedResize(table, free, state, lens, torch.tensor(new, device=dev), PAGE, tokens)

        if tokens == 0:                                               # nobody is left, nobody has come
            have, dense = new, [[None, None] for _ in range(SLOTS)]
            continue
        x = torch.randn((tokens, HIDDEN), device=dev).bfloat16()      # hidden states of all new tokens, request after request
        q, k, v = (layer.project(x, w) for w in (layer.wq, layer.wk, layer.wv))
        blockedAttention.pagedAppend(k, v, layer.k, layer.v, slots, *layer.scales)
        at = {r: sum(grown[:r]) for r in range(SLOTS)}
        if prompts:
            # the prompts' own attention, over segments back to back; key heads are repeated for their query heads.  (It takes the
            # keys and values as the projection gave them, not as a cache in 8 bits has them.)
            rows = torch.cat([torch.arange(at[r], at[r] + new[r]) for r in prompts]).to(dev)
            lengths = torch.tensor([new[r] for r in prompts], device=dev)
            flat = lambda t: t[:, rows].reshape(t.shape[0], -1).contiguous()  # noqa: E731
            wide = lambda t: t.repeat_interleave(GROUP, 0)  # noqa: E731
            inside = blockedAttention.blockFusedAttention(flat(q), flat(wide(k)), flat(wide(v)), lengths, lengths,
                                                          torch.full_like(lengths, DIM), scale=DIM ** -0.5)
            inside = inside.view(HEADS * GROUP, -1, DIM).float().split([new[r] for r in prompts], 1)
            for r, got in zip(prompts, inside):
                qr, kr, vr = (t[:, at[r]:at[r] + new[r]].float() for t in (q, wide(k), wide(v)))
                p = torch.softmax(qr @ kr.transpose(1, 2) * DIM ** -0.5, -1)
                worst = max(worst, (p @ vr - got).abs().max().item())
        # one query per request that has tokens: its newest; ended and empty ones are rows of length 0
        newest = torch.tensor([max(at[r] + grown[r] - 1, 0) for r in range(SLOTS)], device=dev)
        out = blockedAttention.pagedAttention(q[:, newest], layer.k, layer.v, table, lens, scale=DIM ** -0.5,
                                              kScale=layer.scales[0], vScale=layer.scales[1])

        for r in range(SLOTS):
            if new[r] == 0:
                dense[r] = [None, None]
                assert (out[:, r] == 0).all()
                continue
            for i, (t, scale) in enumerate(zip((k, v), layer.scales)):
                mine = t[:, at[r]:at[r] + grown[r]].float()
                if scale is not None:
                    mine = (mine / scale[:, None, None]).clamp(-448, 448).to(torch.float8_e4m3fn).float() * scale[:, None, None]
                dense[r][i] = mine if dense[r][i] is None else torch.cat([dense[r][i], mine], 1)
            qr = q[:, newest[r]].float().view(HEADS, GROUP, DIM)
            p = torch.softmax(qr @ dense[r][0].transpose(1, 2) * DIM ** -0.5, -1)
            worst = max(worst, (p @ dense[r][1] - out[:, r].float().view(HEADS, GROUP, DIM)).abs().max().item())
            answered += 1
        have = new
    assert state[1].item() == 0, f"a step was refused: verdict {state[1].item()}"
    assert lens.tolist() == have
    return worst, answered


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--cache", choices=["bf16", "fp8"], default="bf16")
    parser.add_argument("--steps", type=int, default=40)
    args = parser.parse_args()
    error, count = main(args.cache, args.steps)
    print(f"{count} tokens answered, largest difference from dense attention in fp32: {error:.3g}")
