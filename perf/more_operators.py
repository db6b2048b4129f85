"""Timed cases of drafted and branching answers over a paged key-value cache: a program that answers a batch of requests
by drafting several next tokens at once, or by following several continuations of each request side by side.

A draft is a tree: every drafted token (a node) continues another one of its request or the request's last token.  The
nodes' keys and values are appended to the request's pages behind its other tokens; attention then answers all nodes at
once, the accepted path's tokens move to the front, and the rest is given back.  Rows of the page table that share
what they have read so far share its full pages.  A case is one pass through one of the five operators:

    tree     pagedTree: which nodes each node sees, as bits, and how deep it lies, from every node's parent
    attend   pagedTreeAttention: all nodes of all requests over their caches
    keep     pagedKeep: keys and values of an accepted path move to consecutive places
    fork     pagedFork: rows of the table go on from other rows; pages are shared, the last one is copied, unused ones return
    copy     pagedCopy: pages to other pages

listed() is the fixed list, draw() gives further cases of the same ranges.  The lengths belong to the case (its `sizes`
number seeds them); values, trees, paths and the pages' order come from the seed given to prepare().  With `own` set the
cases call the framework; without it they compute the same with elementary operations in 32 bits.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0


def _tree(requests, nodes, chain=0.3, pad=0, sizes=0):
    """chain: share of nodes that continue the node before them; the others continue any earlier one or the last token."""
    return {"op": "tree", "requests": requests, "nodes": nodes, "chain": chain, "pad": pad, "sizes": sizes}


def _attend(dtype, cache, requests, heads, group, dim, page, lo, hi, nodes, mask="tree", window=0, even=False, flat=False, order="heads", pad=0,
            sizes=0):
    """lo, hi: tokens before the draft; nodes: of a request at most, or of every one (`even`).  mask: "tree", "chain" (every
    node sees those before it) or "any" (a random half of the nodes, some rows none)."""
    return {"op": "attend", "dtype": dtype, "cache": cache, "requests": requests, "heads": heads, "group": group, "dim": dim, "page": page,
            "lo": lo, "hi": hi, "nodes": nodes, "mask": mask, "window": window, "even": even, "flat": flat, "order": order, "pad": pad, "sizes": sizes}


def _keep(dtype, cache, requests, heads, dim, page, hi, nodes, deepest, order="heads", sizes=0):
    """hi: tokens before the draft at most; deepest: entries of a path."""
    return {"op": "keep", "dtype": dtype, "cache": cache, "requests": requests, "heads": heads, "dim": dim, "page": page, "hi": hi,
            "nodes": nodes, "deepest": deepest, "order": order, "sizes": sizes}


def _fork(requests, beams, page, lo, hi, shared=0.5, finish=0.0, sizes=0):
    """Requests of `beams` rows of the table each, which share a part of their pages; a share of the requests ends."""
    return {"op": "fork", "requests": requests, "beams": beams, "page": page, "lo": lo, "hi": hi, "shared": shared, "finish": finish, "sizes": sizes}


def _copy(dtype, cache, copies, heads, dim, page, skip=0.0, order="heads", sizes=0):
    """skip: share of the list's entries that name no page."""
    return {"op": "copy", "dtype": dtype, "cache": cache, "copies": copies, "heads": heads, "dim": dim, "page": page, "skip": skip, "order": order,
            "sizes": sizes}


def listed():
    cases = {
        # One step of a few requests with small drafts.  Launch latency.
        "small_trees": _tree(8, 16),
        # A large batch of deep drafts, most of them long chains; padded rows.
        "deep_trees": _tree(256, 500, chain=0.9, pad=21),
        # A single request with a small draft: latency is all of it.
        "one_tree": _attend("f16", "same", 1, 8, 4, 128, 16, 500, 500, 8, even=True),
        # Ordinary batch with shared heads and drafts of different sizes.
        "tree_batch": _attend("bf16", "same", 32, 8, 4, 128, 16, 1, 4096, 32),
        # Two long documents in an 8-bit cache, token-major pages, large drafts: 512 rows of queries a key head, the largest case.
        "long_trees": _attend("bf16", "fp8", 2, 8, 8, 128, 16, 32768, 65536, 64, even=True, order="tokens"),
        # Guesses without branches, a model without shared heads, an odd head dimension, pages of 24, a sliding window.
        "odd_chain": _attend("f16", "same", 41, 12, 1, 80, 24, 0, 5000, 5, mask="chain", window=1000, flat=True, pad=3),
        # Accepted tokens of an ordinary batch.
        "keep_step": _keep("bf16", "same", 32, 8, 128, 16, 1000, 32, 6),
        # Many requests, deep drafts, a cache in 8 bits whose rows are no whole number of 16 bytes.
        "keep_odd": _keep("f16", "fp8", 200, 5, 100, 24, 500, 120, 40, order="tokens"),
        # Beam search: four continuations of each of eight requests, a step that ends some.
        "beam_fork": _fork(8, 4, 16, 300, 2000, finish=0.1),
        # Many samples of long prompts.
        "wide_fork": _fork(64, 16, 16, 4000, 16000, shared=0.8, finish=0.2),
        # The last pages of those that went on from the same row.
        "copy_tails": _copy("bf16", "same", 32, 8, 128, 16, skip=0.4),
        # Whole prompts: half a gigabyte read and written.
        "copy_prompts": _copy("f16", "same", 4096, 8, 128, 32),
    }
    return [dict(c, name=name) for name, c in cases.items()]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "attend", "attend", "attend", "keep", "fork", "copy"])
    sizes = rng.randrange(1 << 30)
    if op == "tree":
        requests = _log_int(rng, 1, 512)
        nodes = _log_int(rng, 12, min(1000, 130_000 // requests))         # (fewer have hardly any choice of a tree)
        return _tree(requests, nodes, rng.choice([0.0, 0.3, 0.9] if requests * nodes > 100 else [0.0, 0.3]), rng.choice([0, 0, 9]), sizes)
    if op == "fork":
        beams = _log_int(rng, 1, 64)
        hi = _log_int(rng, 1, 16000)
        requests = _log_int(rng, 1, max(2, min(1024, 16_000_000 // hi) // beams))
        return _fork(requests, beams, rng.choice([1, 16, 16, 24, 64, 128]) if hi < 2000 else rng.choice([16, 24, 32, 64, 200]),
                     rng.choice([0, hi // 2, hi]), hi, rng.choice([0.0, 0.5, 0.9]), rng.choice([0.0, 0.2, 0.5]), sizes)
    dtype = rng.choice(["f16", "bf16"])
    cache = rng.choice(["same", "same", "fp8"])
    order = rng.choice(["heads", "heads", "tokens"])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128])
    dim = rng.choice([64, 128, 128, 40, 80, 96, 100, 192, 256, rng.randint(8, 256)])
    heads = _log_int(rng, 1, 16)
    if op == "copy":
        return _copy(dtype, cache, _log_int(rng, 1, max(2, 120_000_000 // (heads * dim * page))), heads, dim, page, rng.choice([0.0, 0.0, 0.5]), order, sizes)
    if op == "keep":
        nodes = _log_int(rng, 2, 200)
        hi = _log_int(rng, 1, 1000)
        requests = _log_int(rng, 1, max(2, min(200, 60_000_000 // (heads * dim * (hi + nodes)))))
        return _keep(dtype, cache, requests, heads, dim, page, hi, nodes, _log_int(rng, 1, min(nodes, 40)), order, sizes)
    group = rng.choice([1, 2, 4, 4, 5, 8, 8, 16])
    hi = _log_int(rng, 1, 65536)
    case = _attend(dtype, cache, _log_int(rng, 1, 128), heads, group, dim, page, rng.choice([0, 1, hi // 3, hi]), hi, _log_int(rng, 1, 256),
                   rng.choice(["tree", "tree", "chain", "any"]), rng.choice([0, 0, 0, _log_int(rng, 1, 8192)]), rng.random() < 0.3,
                   rng.random() < 0.4, order, rng.choice([0, 0, 5]), sizes)
    # no dearer than the largest listed one, nor its rows of scores laid side by side
    most = work(listed()[4])
    while (case["requests"] * heads * group * case["nodes"] * (case["hi"] + case["nodes"]) > 500_000_000
           or case["requests"] * heads * dim * (case["hi"] + case["nodes"]) > 150_000_000 or any(work(case)[k] > most[k] for k in most)):
        if case["requests"] > 1:
            case["requests"] = max(1, case["requests"] * 2 // 3)
        else:
            case["nodes"] = max(1, case["nodes"] * 2 // 3)
            case["hi"] = case["hi"] * 2 // 3
            case["lo"] = min(case["lo"], case["hi"])
    return case


def _pages(lens, page):
    return -(-lens // page)


def _nodes(case, rng):
    """Nodes of every request, the largest draft among them; one request of a ragged batch has none."""
    n, most = case["requests"], case["nodes"]
    if case.get("even"):
        return np.full(n, most, np.int64)
    nodes = rng.integers(1, most + 1, n)
    nodes[rng.integers(n)] = 0
    nodes[rng.integers(n)] = most
    return nodes


def _sizes(case):
    """Tokens before the draft and nodes of every request (`fork`: tokens of every row, of which its request shares the first)."""
    rng = np.random.default_rng(case["sizes"])
    n = case["requests"]
    if case["op"] == "tree":
        return None, _nodes(case, rng)
    if case["op"] == "fork":
        lens = rng.integers(case["lo"], case["hi"] + 1, n)
        shared = np.floor(lens * case["shared"]).astype(np.int64) // case["page"] * case["page"]
        rows = np.repeat(lens, case["beams"])
        some = rng.random(len(rows)) < 0.1                              # rows that ended before the others
        rows = np.where(some, np.maximum(rows - rng.integers(0, 9, len(rows)), np.repeat(shared, case["beams"])), rows)
        return rows, shared
    base = rng.integers(case.get("lo", 0), case["hi"] + 1, n)
    return base, _nodes(case, rng)


def _parents(nodes, chain, gen, dev):
    """A parent for every node of every request: the node before it, or any earlier one (-1: the request's last token)."""
    at = torch.cat([torch.arange(int(n)) for n in nodes]).to(dev) if len(nodes) else torch.zeros(0, dtype=torch.int64, device=dev)
    any_one = (torch.rand(len(at), generator=gen, device=dev) * (at + 1)).long().clamp(max=at) - 1
    return torch.where(torch.rand(len(at), generator=gen, device=dev) < chain, at - 1, any_one)


def _rows_of(accum, longest):
    """For a batch of ragged rows side by side: their places, [requests, longest], and which of them are there."""
    at = accum[:-1, None] + torch.arange(longest, device=accum.device)
    return at, at < accum[1:, None]


def _table(need, extra, gen, dev):
    pages, width = int(need.sum()) + extra, int(need.max()) + 2
    table = torch.full((len(need), width), -1, dtype=torch.int32, device=dev)
    mine = torch.arange(width, device=dev) < torch.from_numpy(need).to(dev)[:, None]
    table[mine] = torch.randperm(pages, generator=gen, device=dev, dtype=torch.int32)[:int(need.sum())]
    return table, pages


def _cache(case, pages, gen, dev):
    """Two arrays of pages, [pages, heads, page, dim], of which either the heads or the tokens follow each other closely."""
    heads, page, dim = case["heads"], case["page"], case["dim"]
    shape = (pages, heads, page, dim) if case["order"] == "heads" else (pages, page, heads, dim)
    got = []
    for _ in range(2):
        t = torch.randn(shape, generator=gen, device=dev, dtype=DTYPES[case["dtype"]])
        if case["cache"] == "fp8":
            t = t.mul_(0.25 * FP8_MAX).clamp_(-FP8_MAX, FP8_MAX).to(FP8)
        got.append(t if case["order"] == "heads" else t.transpose(1, 2))
    return got


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    state = {"op": case["op"]}
    if case["op"] == "copy":
        copies = case["copies"]
        order = torch.randperm(2 * copies + 3, generator=gen, device=dev, dtype=torch.int32)
        skip = torch.rand(copies, generator=gen, device=dev) < case["skip"]
        state.update(source=torch.where(skip, -1, order[:copies]).int(), target=torch.where(skip, -1, order[copies:2 * copies]).int(),
                     cache=_cache(case, 2 * copies + 3, gen, dev))
        return state
    first, second = _sizes(case)
    if case["op"] == "fork":
        beams, page, rows = case["beams"], case["page"], len(first)
        need, common = _pages(first, page), second // page
        used = int(common.sum()) + int((need - np.repeat(common, beams)).sum())
        pages = used + rows + 11
        width = int(need.max()) + 2
        order = torch.randperm(pages, generator=gen, device=dev, dtype=torch.int32)
        column = torch.arange(width, device=dev)
        need, common = (torch.from_numpy(x).to(dev) for x in (need, common))
        shared = common.repeat_interleave(beams)[:, None]
        start = (torch.cumsum(common, 0) - common).repeat_interleave(beams)[:, None]
        alone = need - shared[:, 0]
        own_start = (common.sum() + torch.cumsum(alone, 0) - alone)[:, None]
        at = torch.where(column < shared, start + column, own_start + column - shared)
        table = torch.where(column < need[:, None], order[at.clamp(0, pages - 1)], -1)
        shares = torch.zeros(pages, dtype=torch.int32, device=dev)
        shares[order[:int(common.sum())].long()] = beams - 1
        free = torch.full((pages,), -1, dtype=torch.int32, device=dev)
        free[:pages - used] = order[used:]
        # every row goes on from some row of its request, or its request ends
        family = torch.arange(rows, device=dev) // beams
        origin = family * beams + torch.randint(beams, (rows,), generator=gen, device=dev)
        ends = torch.rand(case["requests"], generator=gen, device=dev) < case["finish"]
        state.update(table=table.int(), free=free, state=torch.tensor([pages - used, 0], device=dev), shares=shares,
                     lens=torch.from_numpy(first).to(dev), origin=torch.where(ends[family], -1, origin), page=page)
        return state
    base, nodes = first, second
    accum = torch.from_numpy(np.concatenate([[0], np.cumsum(nodes)])).to(dev)
    if case["op"] == "tree":
        parents = _parents(nodes, case["chain"], gen, dev)
        pad = torch.full((case["pad"],), -1, dtype=torch.int64, device=dev)
        state.update(parents=torch.cat([parents, pad]), accum=accum, nodes=int(nodes.max()))
        return state
    table, pages = _table(_pages(base + nodes, case["page"]), 5, gen, dev)
    state.update(table=table, cache=_cache(case, pages, gen, dev), base=torch.from_numpy(base).to(dev))
    if case["op"] == "keep":
        # the draft's likeliest chain comes first, its branches behind it: a path follows the chain for a while and then a branch
        deepest = case["deepest"]
        most = torch.from_numpy(np.minimum(nodes, deepest)).to(dev)
        count = (torch.rand(len(most), generator=gen, device=dev) * (most + 1)).long()
        straight = (torch.rand(len(most), generator=gen, device=dev) * (count + 1)).long()[:, None]
        at = torch.arange(deepest, device=dev)
        room = torch.from_numpy(nodes).to(dev) - count                    # branch nodes there are
        branch = count[:, None] + (at - straight) + ((room - count + straight[:, 0]).clamp(min=0).double()
                                                     * torch.rand(len(most), generator=gen, device=dev)).long()[:, None]
        path = torch.where(at < straight, at, torch.where(branch < torch.from_numpy(nodes).to(dev)[:, None], branch, -1))
        state["path"] = torch.where(at < count[:, None], path, -1)
        return state
    tokens, dim = int(nodes.sum()) + case["pad"], case["dim"]
    heads = case["heads"] * case["group"]
    # queries of twice the unit variance: some keys stand out, as in a trained model
    if case["flat"]:
        q = torch.randn((heads, tokens * dim), generator=gen, device=dev)
    else:
        q = torch.randn((tokens, heads, dim), generator=gen, device=dev).transpose(0, 1)
    words = -(-int(nodes.max()) // 64)
    if case["mask"] == "chain":
        mask = None
    elif case["mask"] == "tree":
        parents = torch.cat([_parents(nodes, 0.3, gen, dev), torch.full((case["pad"],), -1, dtype=torch.int64, device=dev)])
        mask = _plain_tree(parents, accum, int(nodes.max()))[0]
    else:
        mask = torch.randint(-2 ** 63, 2 ** 63 - 1, (tokens, words), generator=gen, device=dev)
        mask[torch.rand(tokens, generator=gen, device=dev) < 0.1] = 0
    scales = [None, None]
    if case["cache"] == "fp8":                                            # for values of about unit variance
        scales = [(0.75 + 0.5 * torch.rand(case["heads"], generator=gen, device=dev)) * (4.0 / FP8_MAX) for _ in range(2)]
    state.update(q=(2.0 * q).to(DTYPES[case["dtype"]]), lens=state["base"] + torch.from_numpy(nodes).to(dev), accum=accum, mask=mask,
                 window=case["window"], scale=dim ** -0.5, scales=scales, longest=int((base + nodes).max()), most=int(nodes.max()))
    return state


def run(state):
    s = state
    if own:
        import blockedAttention as ba
    if s["op"] == "tree":
        return (ba.pagedTree if own else _plain_tree)(s["parents"], s["accum"], s["nodes"])
    if s["op"] == "attend":
        if own:
            return ba.pagedTreeAttention(s["q"], *s["cache"], s["table"], s["lens"], s["accum"], s["mask"], scale=s["scale"], window=s["window"],
                                         kScale=s["scales"][0], vScale=s["scales"][1])
        return _plain_attend(s)
    if s["op"] == "keep":
        lens = (ba.pagedKeep if own else _plain_keep)(*s["cache"], s["table"], s["base"], s["path"])
        return [*s["cache"], lens]
    if s["op"] == "fork":
        got = (ba.pagedFork if own else _plain_fork)(s["table"], s["free"], s["state"], s["shares"], s["lens"], s["origin"], s["page"])
        return [*got, s["free"]]
    (ba.pagedCopy if own else _plain_copy)(*s["cache"], s["source"], s["target"])
    return s["cache"]


def _plain_tree(parents, accum, nodes):
    tokens, words = len(parents), max(1, -(-nodes // 64))
    at, there = _rows_of(accum, nodes)
    mine = torch.where(there, at, 0)
    parent = torch.where(there, parents[mine], -1) if tokens else at
    sees = torch.zeros((*at.shape, 64 * words + 1), dtype=torch.bool, device=accum.device)
    node = torch.arange(nodes, device=accum.device).expand(at.shape)
    depth = torch.full(at.shape, -1, device=accum.device)
    for _ in range(nodes):                                                # from every node up to its request's last token
        sees.scatter_(2, torch.where(node >= 0, node, 64 * words)[..., None], True)
        depth = depth + (node >= 0)
        node = torch.where(node >= 0, parent.gather(1, node.clamp(min=0)), -1)
    bits = (sees[..., :-1].reshape(*at.shape, words, 64).long() << torch.arange(64, device=accum.device)).sum(-1)
    mask = torch.zeros((tokens, words), dtype=torch.int64, device=accum.device)
    depths = torch.full((tokens,), -1, device=accum.device)
    mask[at[there]], depths[at[there]] = bits[there], depth[there]
    return mask, depths


def _unpack(mask, words):
    return ((mask[..., None] >> torch.arange(64, device=mask.device)) & 1).bool().reshape(*mask.shape[:-1], 64 * words)


def _sees(s):
    """[requests, nodes, tokens]: what each node's query sees."""
    at, there = _rows_of(s["accum"], s["most"])
    token = torch.arange(s["longest"], device=at.device)
    base, n = s["base"][:, None, None], (s["accum"][1:] - s["accum"][:-1])[:, None, None]
    node = token - base
    inside = (node >= 0) & (node < n)
    if s["mask"] is None:
        own_node = torch.arange(s["most"], device=at.device)[:, None]
        tree = node <= own_node
    else:
        words = s["mask"].shape[1]
        bits = _unpack(s["mask"][torch.where(there, at, 0)], words)
        tree = bits.gather(2, node.clamp(0, 64 * words - 1).expand(-1, s["most"], -1))
    sees = there[..., None] & ((token < base) | (inside & tree))
    if s["window"]:
        rank = sees.flip(2).cumsum(2).flip(2)                             # how many are seen from here on
        sees &= rank <= s["window"]
    return sees, at, there


def _plain_gather(cache, pages, inside, scale):
    if scale is None:
        return cache[pages, :, inside].float()
    return cache.view(torch.uint8)[pages, :, inside].view(FP8).float() * scale[:, None]


def _plain_attend(s):
    kc, vc = s["cache"]
    heads, page, dim = kc.shape[1:]
    sees, at, there = _sees(s)
    tokens = s["q"].reshape(s["q"].shape[0], -1, dim)
    group = tokens.shape[0] // heads
    q = tokens[:, torch.where(there, at, 0)].float()                       # query heads, requests, nodes, dim
    requests, most = at.shape
    q = q.reshape(heads, group, requests, most, dim).permute(2, 0, 1, 3, 4).reshape(requests, heads, group * most, dim)
    token = torch.arange(s["longest"], device=q.device)
    have = token < s["lens"][:, None]
    pages = torch.where(have, s["table"][:, (token // page).clamp(max=s["table"].shape[1] - 1)], 0).long()
    inside = (token % page).expand_as(pages)
    k = _plain_gather(kc, pages, inside, s["scales"][0]).permute(0, 2, 3, 1).contiguous()
    scores = q.matmul(k).reshape(requests, heads, group, most, -1) * s["scale"]
    del k
    scores.masked_fill_(~sees[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = (scores - torch.where(top == -math.inf, 0.0, top)).exp_()
    del scores
    total = p.sum(-1, keepdim=True)
    v = _plain_gather(vc, pages, inside, s["scales"][1]).masked_fill_(~have[:, :, None, None], 0.0).transpose(1, 2).contiguous()
    out = p.reshape(requests, heads, group * most, -1).matmul(v).reshape(requests, heads, group, most, dim)
    out = torch.where(total > 0, out / total, 0.0).permute(1, 2, 0, 3, 4).reshape(heads * group, requests, most, dim)
    result = torch.zeros_like(tokens)
    result[:, at[there]] = out[:, there].to(result.dtype)
    return result.reshape(s["q"].shape)


def _plain_keep(k_cache, v_cache, table, lens, path):
    page = k_cache.shape[2]
    count = (path >= 0).sum(1)
    there = path >= 0
    to = lens[:, None] + torch.arange(path.shape[1], device=path.device)
    row = torch.arange(len(lens), device=path.device)[:, None].expand_as(path)[there]
    to, by = to[there], (lens[:, None] + path)[there]
    pages = [table[row, t // page].long() for t in (to, by)]
    for cache in (k_cache, v_cache):
        cache = cache.view(torch.uint8) if cache.dtype == FP8 else cache
        cache[pages[0], :, to % page] = cache[pages[1], :, by % page]
    return lens + count


def _plain_fork(table, free, state, shares, lens, origin, page):
    rows, width = table.shape
    dev, pages = table.device, len(shares)
    row, column = torch.arange(rows, device=dev), torch.arange(width, device=dev)
    goes = origin >= 0
    by = origin.clamp(min=0)
    children = torch.zeros(rows + 1, dtype=torch.int64, device=dev).index_add_(0, torch.where(goes, by, rows), torch.ones_like(by))[:rows]
    # the last page, where it is not full, stays with the row itself or else with the first that goes on from it
    keeper = torch.full((rows + 1,), rows, device=dev).scatter_reduce_(0, torch.where(goes, by, rows), row, "amin")[:rows]
    keeper = torch.where(origin == row, row, keeper)
    full, part = lens // page, lens % page != 0
    fresh = goes & part[by] & (keeper[by] != row)
    change = torch.where(column < full[:, None], children[:, None] - 1, (children[:, None] > 0).long() - 1)
    change = torch.where(column < (full + part)[:, None], change, 0)
    held = torch.where(column < (full + part)[:, None], table.long(), pages)
    after = torch.cat([shares.long(), shares.new_zeros(1).long()]).index_add_(0, held.reshape(-1), change.reshape(-1))[:pages]
    freed = after < 0
    count, back, taken = state[0], freed.sum(), fresh.sum()
    verdict = (taken > count + back).long() | state[1]
    fine = verdict == 0
    # pages that nobody holds any more, in ascending order, go on the stack; fresh ones come from its end
    given = torch.argsort(~freed, stable=True)
    place = torch.arange(len(free), device=dev)
    stack = torch.where((place >= count) & (place < count + back), given[(place - count).clamp(0, pages - 1)].int(), free)
    number = fresh.cumsum(0) - 1
    target = torch.where(fresh & fine, stack[(count + back - 1 - number).clamp(0, len(free) - 1)], -1)
    last = table[by, full[by].clamp(max=width - 1)]
    source = torch.where(fresh & fine, last, -1)
    new_lens = torch.where(goes, lens[by], 0)
    new_table = torch.where(column < torch.where(goes, (full + part)[by], 0)[:, None], table[by], -1)
    new_table = torch.where((column == full[by][:, None]) & fresh[:, None], target[:, None], new_table)
    left = count + back - taken
    free.copy_(torch.where(fine & (place < left), stack, free))
    return (torch.where(fine, new_table, table), torch.where(fine, new_lens, lens), torch.stack([torch.where(fine, left, count), verdict]),
            torch.where(fine, after.clamp(min=0).int(), shares), source, target)


def _plain_copy(k_cache, v_cache, source, target):
    by, to = source[source >= 0].long(), target[source >= 0].long()
    for cache in (k_cache, v_cache):
        cache = cache.view(torch.uint8) if cache.dtype == FP8 else cache
        cache[to] = cache[by]


def work(case):
    """Bytes that are read or written once, and the products' operations."""
    width = 1 if case.get("cache") == "fp8" else 2
    if case["op"] == "copy":
        return {"bytes": 4 * case["copies"] * case["heads"] * case["page"] * case["dim"] * width * (1 - case["skip"]) + 8 * case["copies"], "flops": 0}
    first, second = _sizes(case)
    if case["op"] == "tree":
        tokens = int(second.sum()) + case["pad"]
        return {"bytes": 8 * (len(second) + 1 + tokens * (2 + -(-case["nodes"] // 64))), "flops": 0}
    if case["op"] == "fork":
        need, common = _pages(first, case["page"]), second // case["page"]
        pages = int(common.sum()) + int((need - np.repeat(common, case["beams"])).sum()) + len(first) + 11
        columns = len(first) * (int(need.max()) + 2)
        # the rows' pages in, the table out; counts of the pages in and out; lengths and origins in, lengths, sources and targets out
        return {"bytes": 4 * (int(need.sum()) + columns + 2 * pages) + 32 * len(first), "flops": 0}
    base, nodes = first, second
    if case["op"] == "keep":
        # half of the deepest path on the average, half of it in place already
        moved = float(np.minimum(nodes, case["deepest"]).sum()) / 4
        return {"bytes": 4 * moved * case["heads"] * case["dim"] * width + 8 * len(base) * (case["deepest"] + 2), "flops": 0}
    seen = np.minimum(base, case["window"]) if case["window"] else base
    seen = np.where(nodes > 0, seen, 0)
    tokens = int((seen + nodes).sum())
    queries = (int(nodes.sum()) + case["pad"]) * case["heads"] * case["group"] * case["dim"]
    words = 0 if case["mask"] == "chain" else -(-case["nodes"] // 64) * int(nodes.sum())
    pages = int(_pages(seen + nodes, case["page"]).sum())
    products = float((nodes * (seen + (nodes + 1) / 2)).sum()) if case["mask"] == "chain" else float((nodes * (seen + 1)).sum())
    return {"bytes": 2 * tokens * case["heads"] * case["dim"] * width + 2 * 2 * queries + 4 * pages + 8 * (2 * len(base) + 1 + words),
            "flops": 4 * products * case["heads"] * case["group"] * case["dim"]}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "copy":
        got = []
        for cache in s["cache"]:
            x = cache.double()
            for a, b in zip(s["source"].tolist(), s["target"].tolist()):
                if a >= 0:
                    x[b] = x[a]
            got.append(x)
        return got
    if case["op"] == "tree":
        # node by node: what the parent sees, and itself
        accum, parents, words = s["accum"].tolist(), s["parents"].tolist(), -(-s["nodes"] // 64)
        sees, depth = [0] * len(parents), [-1] * len(parents)
        for a, b in zip(accum, accum[1:]):
            for i in range(a, b):
                up = a + parents[i] if parents[i] >= 0 else None
                sees[i] = (1 << (i - a)) | (sees[up] if up is not None else 0)
                depth[i] = depth[up] + 1 if up is not None else 0
        mask = np.array([[(x >> (64 * w)) & (2 ** 64 - 1) for w in range(words)] for x in sees], np.uint64).view(np.int64)
        return torch.from_numpy(mask.reshape(len(parents), words)), torch.tensor(depth)
    if case["op"] == "keep":
        got = []
        page, base, path, table = case["page"], s["base"].tolist(), s["path"].tolist(), s["table"].tolist()
        by, to = [], []
        for n, row, mine in zip(base, path, table):
            for i, node in enumerate(row):
                if node >= 0:
                    by.append(mine[(n + node) // page] * page + (n + node) % page)
                    to.append(mine[(n + i) // page] * page + (n + i) % page)
        for cache in s["cache"]:
            x = cache.double().transpose(1, 2).reshape(-1, case["heads"], case["dim"])
            x[to] = x[by]
            got.append(x.reshape(-1, page, case["heads"], case["dim"]).transpose(1, 2))
        return got + [torch.tensor([n + sum(node >= 0 for node in row) for n, row in zip(base, path)])]
    if case["op"] == "fork":
        # row by row, with a list for the stack and a count for every page
        page, lens, origin, table = s["page"], s["lens"].tolist(), s["origin"].tolist(), s["table"].tolist()
        width = len(table[0])
        free, count = s["free"].tolist(), int(s["state"][0])
        holders = [0] * len(s["shares"])
        rows = [row[:_pages(n, page)] for row, n in zip(table, lens)]
        for p in [p for row in rows for p in row]:
            holders[p] += 1
        before = list(holders)
        new, source, target, kept = [], [-1] * len(rows), [-1] * len(rows), set()
        for r, o in enumerate(origin):                                    # a row that goes on from itself keeps its last page
            if o == r:
                kept.add(r)
        copies = []
        for r, o in enumerate(origin):
            row = list(rows[o]) if o >= 0 else []
            if row and lens[o] % page and o != r:
                if o in kept:
                    copies.append(r)
                    row[-1] = -1
                kept.add(o)
            new.append(row)
        holders = [0] * len(holders)
        for p in [p for row in new for p in row if p >= 0]:
            holders[p] += 1
        stack = free[:count] + [p for p in range(len(holders)) if before[p] and not holders[p]]
        for r in copies:
            source[r], target[r] = rows[origin[r]][-1], stack.pop()
            new[r][-1] = target[r]
            holders[target[r]] = 1
        free[count:len(stack)] = stack[count:]
        return (torch.tensor([row + [-1] * (width - len(row)) for row in new], dtype=torch.int32),
                torch.tensor([lens[o] if o >= 0 else 0 for o in origin]), torch.tensor([len(stack), 0]),
                torch.tensor([max(0, h - 1) for h in holders], dtype=torch.int32), torch.tensor(source, dtype=torch.int32),
                torch.tensor(target, dtype=torch.int32), torch.tensor(free, dtype=torch.int32))
    heads, group, dim, page = case["heads"], case["group"], case["dim"], case["page"]
    q = s["q"].double().reshape(heads, group, -1, dim)
    out = torch.zeros_like(q)
    one = [torch.ones(heads, device=q.device)] * 2
    ks, vs = (x.double()[:, None, None] for x in (s["scales"] if case["cache"] == "fp8" else one))
    masks = None if s["mask"] is None else _unpack(s["mask"], s["mask"].shape[1])
    accum = s["accum"].tolist()
    for r, base in enumerate(s["base"].tolist()):
        a, n = accum[r], accum[r + 1] - accum[r]
        if n == 0:
            continue
        sees = torch.ones((n, base + n), dtype=torch.bool, device=q.device)
        sees[:, base:] = torch.ones((n, n), dtype=torch.bool, device=q.device).tril() if masks is None else masks[a:a + n, :n]
        if case["window"]:
            before = sees.sum(1, keepdim=True) - sees.cumsum(1)           # how many of those it sees come later
            sees &= before < case["window"]
        mine = s["table"][r, :_pages(base + n, page)].long()
        k, v = (c.view(torch.uint8)[mine].view(c.dtype) if c.dtype == FP8 else c[mine] for c in s["cache"])
        k, v = (c.double().transpose(0, 1).reshape(heads, -1, dim)[:, :base + n] for c in (k, v))
        for h in range(heads):
            x = torch.matmul(q[h, :, a:a + n], (k[h] * ks[h]).t()) * s["scale"]
            x = torch.where(sees, x, -math.inf)
            p = torch.nan_to_num(torch.softmax(x, -1), nan=0.0)          # (rows that see nothing)
            out[h, :, a:a + n] = torch.matmul(p, v[h] * vs[h])
    return out.reshape(s["q"].shape)
