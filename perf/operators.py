"""Timed cases of the paged key-value cache: what a program does that answers a batch of requests token by token.

The keys and values of every request lie in pages of a fixed number of tokens, in any order; a table gives the pages of a
request in the order of its tokens.  A case is one pass through one of the three operators:

    tables   pagedResize: requests get their new lengths; pages change hands, new tokens get their places
    append   pagedAppend: keys and values of new tokens are written to their places, in 16 bits or rounded to 8 (e4m3)
    attend   pagedAttention: one query per request and head over the request's whole cache or the window's part of it

listed() is the fixed list, draw() gives further cases of the same ranges.  The lengths belong to the case (its `sizes`
number seeds them); values and the pages' order come from the seed given to prepare().  With `own` set the cases call the
framework; without it they compute the same with elementary operations in 32 bits.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0


def _tables(requests, page, width, lo, hi, one=1.0, prompt=0.0, finish=0.0, back=0.0, pad=0, sizes=0):
    """Shares of the requests that get one more token, arrive with a prompt, end, and lose up to eight tokens again."""
    return {"op": "tables", "requests": requests, "page": page, "width": width, "lo": lo, "hi": hi, "one": one, "prompt": prompt,
            "finish": finish, "back": back, "pad": pad, "sizes": sizes}


def _append(dtype, cache, tokens, heads, dim, page, flat, order="heads", pad=0, sizes=0):
    return {"op": "append", "dtype": dtype, "cache": cache, "tokens": tokens, "heads": heads, "dim": dim, "page": page, "flat": flat,
            "order": order, "pad": pad, "sizes": sizes}


def _attend(dtype, cache, requests, heads, group, dim, page, lo, hi, skew=1.0, window=0, empty=0, flat=False, order="heads", sizes=0):
    return {"op": "attend", "dtype": dtype, "cache": cache, "requests": requests, "heads": heads, "group": group, "dim": dim, "page": page,
            "lo": lo, "hi": hi, "skew": skew, "window": window, "empty": empty, "flat": flat, "order": order, "sizes": sizes}


def listed():
    cases = {
        # A step of a full batch: every request gets one token, a few of them a page.  Launch latency.
        "step_tables": _tables(256, 16, 512, 1, 8000),
        # A batch of prompts arrives in an empty cache: hundreds of thousands of places.
        "prompt_tables": _tables(64, 64, 128, 0, 0, one=0.0, prompt=1.0),
        # Many requests at all stages at once, some rejected draft tokens; a page size that is no power of two; padded slots.
        "mixed_tables": _tables(2000, 24, 100, 1, 2300, one=0.75, prompt=0.02, finish=0.13, back=0.1, pad=37),
        # The keys and values of one step of 64 requests, from the rows of a projection.
        "step_append": _append("bf16", "same", 64, 8, 128, 16, flat=False, pad=3),
        # Prompts of a batch, in the layout that the attention over prompts takes.
        "prompt_append": _append("f16", "same", 16384, 8, 128, 16, flat=True),
        # Prompts into a cache in 8 bits; token-major pages, an odd number of tokens.
        "fp8_append": _append("bf16", "fp8", 30011, 8, 64, 32, flat=False, order="tokens"),
        # A single request: latency is all of it.
        "one_request": _attend("f16", "same", 1, 8, 4, 128, 16, 500, 500),
        # Ordinary batch with shared heads; a few empty rows that pad the batch to a fixed size.
        "batch": _attend("bf16", "same", 64, 8, 4, 128, 16, 1, 4096, empty=3),
        # Few requests over very long documents: the cache's length has to be split.
        "long_few": _attend("f16", "same", 3, 8, 8, 128, 64, 40000, 131072),
        # The largest batch, lengths far apart: memory traffic is all of it.
        "large_batch": _attend("bf16", "same", 128, 8, 4, 128, 32, 1, 16384, skew=1.5),
        # Cache in 8 bits, eight query heads to a key head, token-major pages.
        "fp8_batch": _attend("bf16", "fp8", 96, 8, 8, 128, 16, 1, 8192, order="tokens"),
        # A model without shared heads, an odd head dimension, pages of 24, a sliding window.
        "odd_window": _attend("f16", "same", 41, 12, 1, 80, 24, 1, 5000, window=1000, flat=True),
    }
    return [dict(c, name=name) for name, c in cases.items()]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tables", "append", "attend", "attend"])
    sizes = rng.randrange(1 << 30)
    if op == "tables":
        page = rng.choice([1, 8, 16, 16, 24, 32, 64, 128, 200])
        longest = _log_int(rng, 4 * page, 8192)
        requests = _log_int(rng, 1, max(2, min(4096, 4_000_000 // longest)))
        one, prompt, finish, back = rng.choice([(1.0, 0.0, 0.0, 0.0), (0.0, 1.0, 0.0, 0.0), (0.6, 0.1, 0.2, 0.1), (0.2, 0.02, 0.08, 0.7)])
        if prompt > 0.5:
            requests = min(requests, max(1, 500_000 // longest))
        return _tables(requests, page, -(-longest // page) + rng.choice([0, 1, 13]), 0 if prompt > 0.5 else 1,
                       0 if prompt > 0.5 else max(1, longest - 1), one, prompt, finish, back, rng.choice([0, 0, 5, 100]), sizes)
    dtype = rng.choice(["f16", "bf16"])
    cache = rng.choice(["same", "same", "fp8"])
    order = rng.choice(["heads", "heads", "tokens"])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128, 256])
    dim = rng.choice([64, 128, 128, 40, 80, 96, 100, 192, 256, rng.randint(8, 256)])
    flat = rng.random() < 0.4
    if op == "append":
        heads = _log_int(rng, 1, 32)
        tokens = _log_int(rng, 1, max(2, 30_000_000 // (heads * dim)))
        return _append(dtype, cache, tokens, heads, dim, page, flat, order, rng.choice([0, 0, 7]), sizes)
    heads = _log_int(rng, 1, 16)
    group = rng.choice([1, 2, 4, 5, 8, 8, 16, 24, 32])
    hi = _log_int(rng, 1, 131072)
    lo = rng.choice([1, 1, max(1, hi // 3), hi])
    requests = _log_int(rng, 1, 256)
    case = _attend(dtype, cache, requests, heads, group, dim, page, lo, hi, rng.choice([1.0, 1.0, 3.0]),
                   rng.choice([0, 0, 0, _log_int(rng, 1, 8192)]), 0, flat, order, sizes)
    # no dearer than the largest listed one, nor its lengths laid side by side
    most = work(listed()[9])
    while case["requests"] * case["hi"] * case["heads"] * dim > 128 * 16384 * 1024 or any(work(case)[k] > most[k] for k in most):
        if case["requests"] > 1:
            case["requests"] = max(1, case["requests"] * 2 // 3)
        else:
            case["heads"] = max(1, case["heads"] // 2)
    if case["requests"] > 4:
        case["empty"] = rng.choice([0, 1, 2])
    return case


def _lengths(case):
    """Lengths of the requests of an `attend` case, before and after the call of a `tables` case."""
    rng = np.random.default_rng(case["sizes"])
    n = case["requests"]
    if case["op"] == "attend":
        lens = case["lo"] + np.floor((case["hi"] - case["lo"] + 1) * rng.random(n) ** case["skew"]).astype(np.int64)
        lens = np.minimum(lens, case["hi"])
        lens[rng.permutation(n)[:case["empty"]]] = 0
        return lens
    most = case["page"] * case["width"]
    old = rng.integers(case["lo"], case["hi"] + 1, n)
    kind = rng.choice(4, n, p=np.array([case["one"], case["prompt"], case["finish"], case["back"]]))
    old[kind == 1] = 0
    new = np.select([kind == 0, kind == 1, kind == 2], [old + 1, rng.integers(1, most + 1, n), 0 * old],
                    np.maximum(old - rng.integers(1, 9, n), 0))
    return old, np.minimum(new, most)


def _pages(lens, page):
    return -(-lens // page)


def _cache(case, pages, gen, dev):
    """Two arrays of pages, [pages, heads, page, dim], of which either the heads or the tokens follow each other closely."""
    heads, page, dim = case["heads"], case["page"], case["dim"]
    shape = (pages, heads, page, dim) if case["order"] == "heads" else (pages, page, heads, dim)
    got = []
    for _ in range(2):
        t = torch.randn(shape, generator=gen, device=dev, dtype=DTYPES[case["dtype"]])
        if case["cache"] == "fp8":
            t = t.mul_(0.25 * FP8_MAX).clamp_(-FP8_MAX, FP8_MAX).to(FP8)      # one value in 16000 at the limit
        got.append(t if case["order"] == "heads" else t.transpose(1, 2))
    return got


def _scales(case, gen, dev):
    """What the stored values of each head are multiplied with, for values of about unit variance."""
    if case["cache"] != "fp8":
        return None, None
    return [(0.75 + 0.5 * torch.rand(case["heads"], generator=gen, device=dev)) * (4.0 / FP8_MAX) for _ in range(2)]


def _rows(case, heads, rows, gen, dev, factor=1.0):
    """[heads, rows * dim], or rows of a projection seen as [heads, rows, dim]."""
    if case["flat"]:
        t = torch.randn((heads, rows * case["dim"]), generator=gen, device=dev)
    else:
        t = torch.randn((rows, heads, case["dim"]), generator=gen, device=dev).transpose(0, 1)
    return (t * factor).to(DTYPES[case["dtype"]])


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    state = {"op": case["op"], "page": case["page"]}
    if case["op"] == "tables":
        old, new = _lengths(case)
        o, n = _pages(old, case["page"]), _pages(new, case["page"])
        held, pool = int(o.sum()), int(o.sum() + np.maximum(n - o, 0).sum()) + 17
        order = torch.randperm(pool, generator=gen, device=dev, dtype=torch.int32)
        table = torch.full((case["requests"], case["width"]), -1, dtype=torch.int32, device=dev)
        mine = torch.arange(case["width"], device=dev) < torch.from_numpy(o).to(dev)[:, None]
        table[mine] = order[:held]
        free = torch.full((pool,), -1, dtype=torch.int32, device=dev)
        free[:pool - held] = order[held:]
        state.update(table=table, free=free, state=torch.tensor([pool - held, 0], device=dev), lens=torch.from_numpy(old).to(dev),
                     new=torch.from_numpy(new).to(dev), tokens=int(np.maximum(new - old, 0).sum()) + case["pad"])
        return state
    state["scales"] = _scales(case, gen, dev)
    if case["op"] == "append":
        pages = _pages(case["tokens"], case["page"]) + 9
        places = torch.randperm(pages, generator=gen, device=dev)[:, None] * case["page"] + torch.arange(case["page"], device=dev)
        slots = places.reshape(-1)[:case["tokens"]].contiguous()              # page by page, the pages in any order
        slots[case["tokens"] - min(case["pad"], case["tokens"] - 1):] = -1     # rows that pad the batch
        state.update(slots=slots, k=_rows(case, case["heads"], case["tokens"], gen, dev),
                     v=_rows(case, case["heads"], case["tokens"], gen, dev), cache=_cache(case, pages, gen, dev))
        return state
    lens = _lengths(case)
    need = _pages(lens, case["page"])
    pages, width = int(need.sum()) + 5, int(need.max()) + 3
    table = torch.full((case["requests"], width), -1, dtype=torch.int32, device=dev)
    mine = torch.arange(width, device=dev) < torch.from_numpy(need).to(dev)[:, None]
    table[mine] = torch.randperm(pages, generator=gen, device=dev, dtype=torch.int32)[:int(need.sum())]
    # queries of twice the unit variance: some keys stand out, as in a trained model
    state.update(table=table, lens=torch.from_numpy(lens).to(dev), longest=int(lens.max()), window=case["window"],
                 q=_rows(case, case["heads"] * case["group"], case["requests"], gen, dev, 2.0), scale=case["dim"] ** -0.5,
                 cache=_cache(case, pages, gen, dev))
    return state


def run(state):
    s = state
    if s["op"] == "tables":
        if own:
            import blockedAttention
            got = blockedAttention.pagedResize(s["table"], s["free"], s["state"], s["lens"], s["new"], s["page"], s["tokens"])
        else:
            got = _plain_tables(**{k: v for k, v in s.items() if k != "op"})
        return [*got, s["table"], s["free"]]
    if s["op"] == "append":
        if own:
            import blockedAttention
            blockedAttention.pagedAppend(s["k"], s["v"], *s["cache"], s["slots"], *s["scales"])
        else:
            _plain_append(s["k"], s["cache"][0], s["slots"], s["scales"][0])
            _plain_append(s["v"], s["cache"][1], s["slots"], s["scales"][1])
        return s["cache"]
    if own:
        import blockedAttention
        return blockedAttention.pagedAttention(s["q"], *s["cache"], s["table"], s["lens"], scale=s["scale"], window=s["window"],
                                               kScale=s["scales"][0], vScale=s["scales"][1])
    return _plain_attend(s)


def _plain_tables(table, free, state, lens, new, page, tokens):
    width, dev = table.shape[1], table.device
    count, columns = state[0], torch.arange(table.shape[1], device=table.device)
    o, n = (lens + page - 1) // page, (new + page - 1) // page
    take, drop, grow = (n - o).clamp(min=0), (o - n).clamp(min=0), (new - lens).clamp(min=0)
    taken, dropped = take.cumsum(0), drop.cumsum(0)
    accum = torch.cat([grow.new_zeros(1), grow.cumsum(0)])
    verdict = ((taken[-1] > count + dropped[-1]).long() + 2 * (n > width).any() + 4 * ((lens < 0) | (new < 0)).any()
               + 8 * (accum[-1] > tokens)) | state[1]
    fine = verdict == 0
    # pages that are given back, in order of requests and columns
    back = (columns >= n[:, None]) & (columns < o[:, None])
    number = torch.where(back, (dropped - drop)[:, None] + columns - n[:, None], table.numel())
    given = table.new_zeros(table.numel() + 1).scatter_(0, number.reshape(-1), table.reshape(-1))
    # pages that are taken: first those, then the free ones from the end
    fresh = (columns >= o[:, None]) & (columns < n[:, None]) & fine
    number = (taken - take)[:, None] + columns - o[:, None]
    rest = (count - 1 - (number - dropped[-1])).clamp(0, free.numel() - 1)
    page_of = torch.where(number < dropped[-1], given[number.clamp(0, table.numel())], free[rest])
    place = torch.arange(free.numel(), device=dev)
    number = (count + dropped[-1] - 1 - place).clamp(0, table.numel())
    free.copy_(torch.where((place >= count) & (place < count + dropped[-1] - taken[-1]) & fine, given[number], free))
    table.copy_(torch.where(fresh, page_of, table))
    token = torch.arange(tokens, device=dev)
    row = torch.searchsorted(accum[1:], token, right=True).clamp(max=lens.numel() - 1)
    at = lens[row] + token - accum[row]
    slots = table[row, (at // page).clamp(0, width - 1)].long() * page + at % page
    slots = torch.where((token < accum[-1]) & fine, slots, -1)
    after = torch.stack([torch.where(fine, count + dropped[-1] - taken[-1], count), verdict])
    return slots, accum, torch.where(fine, new, lens), after


def _plain_append(x, cache, slots, scale):
    page, dim = cache.shape[2:]
    rows = x.reshape(x.shape[0], -1, dim).transpose(0, 1)[slots >= 0]
    at = slots[slots >= 0]
    if scale is not None:
        rows = (rows.float() / scale[:, None]).clamp(-FP8_MAX, FP8_MAX).to(FP8).view(torch.uint8)
        cache = cache.view(torch.uint8)
    cache[at // page, :, at % page] = rows


def _plain_gather(cache, pages, inside, scale):
    if scale is None:
        return cache[pages, :, inside].float()
    return cache.view(torch.uint8)[pages, :, inside].view(FP8).float() * scale[:, None]


def _plain_attend(s):
    kc, vc = s["cache"]
    heads, page, dim = kc.shape[1:]
    q = s["q"].reshape(s["q"].shape[0], -1, dim).float()
    q = q.reshape(heads, -1, *q.shape[1:]).permute(2, 0, 1, 3)                  # requests, key heads, group, dim
    at = torch.arange(s["longest"], device=q.device)
    there = at < s["lens"][:, None]
    if s["window"]:
        there &= at >= s["lens"][:, None] - s["window"]
    pages = torch.where(there, s["table"][:, at // page], 0).long()
    inside = (at % page).expand_as(pages)
    k = _plain_gather(kc, pages, inside, s["scales"][0]).permute(0, 2, 3, 1)     # requests, heads, dim, tokens
    scores = torch.where(there[:, None, None], q.matmul(k) * s["scale"], -math.inf)
    del k
    most = scores.amax(-1, keepdim=True)
    p = (scores - torch.where(there.any(-1)[:, None, None, None], most, 0.0)).exp()
    v = _plain_gather(vc, pages, inside, s["scales"][1]).masked_fill_(~there[:, :, None, None], 0.0).transpose(1, 2)
    out = p.matmul(v) / p.sum(-1, keepdim=True)
    out = torch.where(there.any(-1)[:, None, None, None], out, 0.0)
    out = out.permute(1, 2, 0, 3).reshape(-1, len(pages), dim).to(s["q"].dtype)
    return out.reshape(s["q"].shape)


def work(case):
    """Bytes that are read or written once, and the products' operations."""
    if case["op"] == "tables":
        old, new = _lengths(case)
        o, n = _pages(old, case["page"]), _pages(new, case["page"])
        take, drop = int(np.maximum(n - o, 0).sum()), int(np.maximum(o - n, 0).sum())
        tokens = int(np.maximum(new - old, 0).sum()) + case["pad"]
        # lengths before and after, prefix sums and lengths out, places; pages read and written
        return {"bytes": 8 * (4 * len(old) + 1 + tokens) + 4 * (2 * take + drop + max(drop - take, 0)), "flops": 0}
    width = 1 if case["cache"] == "fp8" else 2
    if case["op"] == "append":
        rows = case["tokens"] - min(case["pad"], case["tokens"] - 1)
        return {"bytes": 2 * rows * case["heads"] * case["dim"] * (2 + width) + 8 * case["tokens"], "flops": 0}
    lens = _lengths(case)
    seen = np.minimum(lens, case["window"]) if case["window"] else lens
    tokens, pages = int(seen.sum()), int((_pages(lens, case["page"]) - (lens - seen) // case["page"]).sum())
    queries = case["requests"] * case["heads"] * case["group"] * case["dim"]
    return {"bytes": 2 * tokens * case["heads"] * case["dim"] * width + 2 * 2 * queries + 4 * pages + 8 * len(lens),
            "flops": 4 * tokens * case["heads"] * case["group"] * case["dim"]}


def _e4m3(x):
    """The nearest number of four significand bits, ties to even, steps of 2^-9 at the least, at most 448."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-FP8_MAX, FP8_MAX)


def exact(case, seed):
    s = prepare(case, seed)
    page = s["page"]
    if case["op"] == "tables":
        # request by request, with a list for the stack
        old, new, table, free = (s[k].tolist() for k in ("lens", "new", "table", "free"))
        count = int(s["state"][0])
        stack, given, slots, accum = free[:count], [], [], [0]
        for a, b, row in zip(old, new, table):
            given += row[_pages(b, page):_pages(a, page)]
        stack += given[::-1]
        for a, b, row in zip(old, new, table):
            for column in range(_pages(a, page), _pages(b, page)):
                row[column] = stack.pop()
            slots += [row[t // page] * page + t % page for t in range(a, b)]
            accum.append(len(slots))
        free[count:len(stack)] = stack[count:]
        slots += [-1] * (s["tokens"] - len(slots))
        return [torch.tensor(x) for x in (slots, accum, new, [len(stack), 0])] + [torch.tensor(x, dtype=torch.int32) for x in (table, free)]
    if case["op"] == "append":
        got = []
        for x, cache, scale in zip((s["k"], s["v"]), s["cache"], s["scales"]):
            x = x.double().reshape(case["heads"], case["tokens"], case["dim"])
            if scale is not None:
                x = _e4m3(x / scale.double()[:, None, None])
            flat = cache.double().transpose(1, 2).reshape(-1, case["heads"], case["dim"])
            for h in range(case["heads"]):
                flat[s["slots"][s["slots"] >= 0], h] = x[h, s["slots"] >= 0]
            got.append(flat.reshape(-1, page, *flat.shape[1:]).transpose(1, 2))
        return got
    q = s["q"].double().reshape(case["heads"], case["group"], case["requests"], case["dim"])
    out = torch.zeros_like(q)
    one = [torch.ones(case["heads"], device=q.device)] * 2
    ks, vs = (x.double()[:, None, None] for x in (s["scales"] if case["cache"] == "fp8" else one))
    for r, n in enumerate(s["lens"].tolist()):
        if n:
            first = max(0, n - case["window"]) if case["window"] else 0
            mine = s["table"][r, :_pages(n, page)].long()
            k, v = (c.view(torch.uint8)[mine].view(c.dtype) if c.dtype == FP8 else c[mine] for c in s["cache"])
            k, v = (c.double().transpose(0, 1).reshape(case["heads"], -1, case["dim"])[:, first:n] for c in (k, v))
            p = torch.softmax(torch.matmul(q[:, :, r], (k * ks).transpose(1, 2)) * s["scale"], -1)
            out[:, :, r] = torch.matmul(p, v * vs)
    return out.reshape(s["q"].shape)
