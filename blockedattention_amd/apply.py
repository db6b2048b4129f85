"""Python surface of the operators: the reference's ``blockGEMM`` and
``blockSoftmax`` (blockedAttention/apply.py:6-41) with identical names,
argument order and defaults, plus the fused pair.

All three forward to the compiled extension ``blockAttention`` (built in-tree
by ``python -m blockedattention_amd.build``); there is no Python or CPU
fallback.  The reference wrapper passes ``srcAccum`` to the extension in the
wrong position (apply.py:41 against csrc/sparseBlockedAttention.cpp:127-128);
here the call follows the extension's order, so ``blockSoftmax(x, rows, cols)``
works as documented.
"""
from typing import Optional, Tuple

import torch

from . import blockAttention


def blockGEMM(
    mat1: torch.Tensor, mat2: torch.Tensor,
    mat1Accum: Optional[torch.Tensor] = None, mat2Accum: Optional[torch.Tensor] = None,
    outAccum: Optional[torch.Tensor] = None,
    MList: Optional[torch.Tensor] = None, NList: Optional[torch.Tensor] = None, KList: Optional[torch.Tensor] = None,
    transpose1: Optional[bool] = False, transpose2: Optional[bool] = False,
) -> torch.Tensor:
    """Varlen GEMM ``out_g = A_g @ B_g^T`` over segments stored back to back.

    ``mat1`` is ``[H, sum(M_g*K_g)]``, ``mat2`` is ``[H, sum(N_g*K_g)]`` and the
    result ``[H, sum(M_g*N_g)]``; segment ``g`` is row-major ``M_g x K_g``
    (``K_g x M_g`` with ``transpose1``), ``N_g x K_g`` (``K_g x N_g`` with
    ``transpose2``) and ``M_g x N_g``.  Give either the three exclusive prefix
    sums (int64, one more entry than segments) or the three size lists (int64),
    or both.
    """
    return blockAttention.sparseBlockedGEMM(mat1, mat2, mat1Accum, mat2Accum, outAccum, MList, NList, KList,
                                            bool(transpose1), bool(transpose2))


def blockSoftmax(
    src: torch.Tensor,
    rowList: torch.Tensor, colList: torch.Tensor, srcAccum: Optional[torch.Tensor] = None,
    scale: float = 1.0,
) -> torch.Tensor:
    """Row softmax inside every ``rowList[g] x colList[g]`` block of ``src`` (``[H, sum(rows*cols)]``).

    ``srcAccum`` (the exclusive prefix sum of ``rows*cols``) is optional.
    ``scale`` multiplies the input first; the default 1.0 is the reference's
    behaviour.
    """
    if scale == 1.0:
        return blockAttention.sparseBlockedSoftmax(src, rowList, colList, srcAccum)
    return blockAttention.sparseBlockedSoftmaxScaled(src, rowList, colList, srcAccum, float(scale))


def blockGEMMSoftmax(
    mat1: torch.Tensor, mat2: torch.Tensor,
    mat1Accum: Optional[torch.Tensor] = None, mat2Accum: Optional[torch.Tensor] = None,
    outAccum: Optional[torch.Tensor] = None,
    MList: Optional[torch.Tensor] = None, NList: Optional[torch.Tensor] = None, KList: Optional[torch.Tensor] = None,
    scale: float = 1.0, out_fp32: bool = False,
) -> torch.Tensor:
    """Fused ``softmax(scale * A_g @ B_g^T)`` per segment (forward only).

    Same operands and metadata as ``blockGEMM`` (untransposed layouts); the
    scores stay in fp32 registers between the product and the softmax, so the
    result is what ``blockSoftmax(blockGEMM(...), MList, NList, scale=scale)``
    computes without the intermediate 16-bit rounding.
    """
    return blockAttention.sparseBlockedGEMMSoftmax(mat1, mat2, mat1Accum, mat2Accum, outAccum, MList, NList, KList,
                                                   float(scale), bool(out_fp32))


def blockFusedAttention(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
    MList: Optional[torch.Tensor] = None, NList: Optional[torch.Tensor] = None, KList: Optional[torch.Tensor] = None,
    mat1Accum: Optional[torch.Tensor] = None, mat2Accum: Optional[torch.Tensor] = None,
    outAccum: Optional[torch.Tensor] = None,
    scale: float = 1.0,
) -> torch.Tensor:
    """``softmax(scale * Q_g @ K_g^T) @ V_g`` per segment in one pass.

    ``q`` is ``[H, sum(M*K)]`` (the first operand of ``blockGEMM``), ``k`` and ``v`` are both
    ``[H, sum(N*K)]`` (its second operand's layout); the metadata is ``blockGEMM``'s.  The result,
    ``[H, sum(M*K)]``, is what ``blockGEMM(blockSoftmax(blockGEMM(q, k, ...), M, N, scale=scale), v, ...,
    transpose2=True)`` computes, without the ``M x N`` arrays ever reaching memory.  Head dimensions up
    to 128.  Differentiable in q, k and v when the size lists are given: the forward pass then also keeps one
    number per query, from which the backward kernels recompute the probabilities.
    """
    return blockAttention.sparseBlockedAttention(q, k, v, mat1Accum, mat2Accum, outAccum, MList, NList, KList,
                                                 float(scale))


def pagedResize(
    table: torch.Tensor, free: torch.Tensor, state: torch.Tensor,
    lens: torch.Tensor, newLens: torch.Tensor, pageSize: int, tokens: int,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Request ``r`` goes from ``lens[r]`` to ``newLens[r]`` tokens: pages change hands, new tokens get places.

    ``table`` (int32 ``[requests, width]``) holds every request's pages in the order of its tokens, ``free`` (int32) is a
    stack whose first ``state[0]`` entries are the free pages; both are updated in place.  ``state`` is int64 ``[2]``:
    that count and 0.  Lengths (int64) of 0 are requests that are not there.  Pages are taken in the order of requests,
    first those that shrinking requests give back, then the free ones from the end of the stack.

    Returns ``(slots, tokenAccum, lens, state)``: the places (``page * pageSize + row``, int64 ``[tokens]``) of the new
    tokens, request after request, then -1; their exclusive prefix sums per request; the new lengths; the new state.
    ``tokens`` is at least the number of new tokens.  Where there are too few pages, slots or entries in a row, or a
    length is not valid, nothing changes hands, all slots are -1, the lengths come back as they were and ``state[1]`` is
    a sum of 1 (too few pages), 2 (row too short), 4 (bad length), 8 (more new tokens than ``tokens``), 16 (bad
    state).  A state with a verdict is refused again, so it may be looked at many steps later; nothing synchronises with
    the host.
    """
    return tuple(blockAttention.pagedResize(table, free, state, lens, newLens, int(pageSize), int(tokens)))


def pagedAppend(
    k: torch.Tensor, v: torch.Tensor, kCache: torch.Tensor, vCache: torch.Tensor, slots: torch.Tensor,
    kScale: Optional[torch.Tensor] = None, vScale: Optional[torch.Tensor] = None,
) -> None:
    """Writes the keys and values of new tokens to their places (``slots``, of ``pagedResize``) in a paged cache.

    ``k`` and ``v`` are ``[heads, tokens * dim]`` (the layout of ``blockFusedAttention``) or ``[heads, tokens, dim]`` with any
    strides of heads and tokens, the caches ``[pages, heads, page, dim]`` with any strides but the last.  The caches have
    the dtype of ``k`` and ``v`` (fp16 or bf16), or are ``float8_e4m3fn``: then ``kScale`` and ``vScale`` (fp32
    ``[heads]``) are what stored values are multiplied with; values are divided by it in fp32, limited to +-448 and
    the quotient is rounded to the nearest, ties to even.  Places below 0 are skipped; no place may occur twice.
    """
    blockAttention.pagedAppend(k, v, kCache, vCache, slots, kScale, vScale)


def pagedAttention(
    q: torch.Tensor, kCache: torch.Tensor, vCache: torch.Tensor, table: torch.Tensor, lens: torch.Tensor,
    scale: float = 1.0, window: int = 0,
    kScale: Optional[torch.Tensor] = None, vScale: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """``softmax(scale * q K^T) V`` of one query per request and head over the request's tokens in a paged cache.

    ``q`` is ``[heads, requests * dim]`` or ``[heads, requests, dim]`` with any strides of heads and requests; its heads
    are a multiple of the cache's, consecutive ones share a key head.  ``table`` and ``lens`` are those of
    ``pagedResize`` (here a table may also be one row expanded over the requests), the caches and scales those of
    ``pagedAppend``.  ``window`` > 0 looks at the last ``window`` tokens only.  Requests of length 0 give zeros.  The result
    has the shape, dtype and order of dimensions of ``q`` (contiguous where rows of ``q`` overlap so that they have no
    order).  Forward only; nothing synchronises with the host.
    """
    return blockAttention.pagedAttention(q, kCache, vCache, table, lens, float(scale), int(window), kScale, vScale)


def pagedTree(parents: torch.Tensor, accum: torch.Tensor, nodes: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """What the nodes of trees of drafted tokens see, and how deep they lie.

    The nodes of request ``r`` are rows ``accum[r] .. accum[r + 1] - 1`` (int64, the ``tokenAccum`` of ``pagedResize``);
    ``parents`` (int64, one entry a row) is the number of a node's parent within its request, which comes before it, or -1 for
    the request's last token.  ``nodes`` (up to 1024) is the most that a request has.

    Returns ``(mask, depth)``: int64 ``[rows, words]`` with bit ``j % 64`` of word ``j // 64`` set where the row's node goes
    on from node ``j`` of its request or is it, and int64 ``[rows]``, the number of nodes it goes on from (so a node's
    position is the request's length before the draft plus its depth).  Rows of no request, nodes beyond ``nodes`` and
    nodes whose parent, or a parent's parent, does not come before its node get no bits and depth -1.
    """
    return tuple(blockAttention.pagedTree(parents, accum, int(nodes)))


def pagedTreeAttention(
    q: torch.Tensor, kCache: torch.Tensor, vCache: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, accum: torch.Tensor,
    mask: Optional[torch.Tensor] = None, scale: float = 1.0, window: int = 0,
    kScale: Optional[torch.Tensor] = None, vScale: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """``pagedAttention`` for several queries of a request: of all nodes of a tree of drafted tokens, or of a piece of a prompt.

    ``q`` is ``[heads, tokens * dim]`` or ``[heads, tokens, dim]``; request ``r`` has its rows ``accum[r] .. accum[r + 1] - 1``,
    whose keys and values are the last of its ``lens[r]`` tokens in the cache (``tokenAccum`` and ``lens`` as ``pagedResize``
    returns them).  A row sees all tokens before those and, of those, the ones whose bits its row of ``mask`` has (int64
    ``[tokens, words]``, of ``pagedTree`` or any other); without a mask those before it and itself.  ``window`` > 0 looks at the
    last ``window`` tokens that a row sees.  Rows that see nothing, or whose scores are all -infinity, give zeros, and so do rows of no request; what a
    row does not see has no influence on it.  All else is as for ``pagedAttention``.
    """
    return blockAttention.pagedTreeAttention(q, kCache, vCache, table, lens, accum, mask, float(scale), int(window), kScale, vScale)


def pagedKeep(kCache: torch.Tensor, vCache: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, path: torch.Tensor) -> torch.Tensor:
    """Moves the keys and values of accepted nodes to the front of their draft, in place.

    ``lens`` (int64) are the requests' lengths before the draft, ``path`` (int64 ``[requests, depth]``) the accepted nodes in
    their order, then -1: the token at ``lens[r] + path[r, i]`` comes to ``lens[r] + i``.  A path increases; it ends at the first entry
    that does not, is below its own index, or lies outside the row.  Returns the lengths with the accepted nodes; ``pagedResize``
    to those gives the other pages back.  Call it for every layer's cache.  Pages that are written must not be another row's
    too (``pagedFork`` sees to that), so a draft whose step ``pagedResize`` refused keeps nothing: ``torch.where(state[1] == 0,
    path, -1)`` as the path.
    """
    return blockAttention.pagedKeep(kCache, vCache, table, lens, path)


def pagedFork(
    table: torch.Tensor, free: torch.Tensor, state: torch.Tensor, shares: torch.Tensor, lens: torch.Tensor, origin: torch.Tensor, pageSize: int,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Row ``r`` of the table goes on from row ``origin[r]``: itself, another one whose tokens it has from then on, or -1 if it ends.

    ``table``, ``free``, ``state`` and ``lens`` are those of ``pagedResize``; ``shares`` (int32, an entry for each page of the cache, zeros at
    first) counts the rows that hold a page beyond the first.  Full pages are shared.  A last page that is not full stays
    with the row itself if it goes on, else with the first row that goes on from it; the others get a fresh page each.  Pages that no row
    holds any more go on the stack in ascending order, before fresh ones are taken from its end.  ``free`` is updated in
    place.

    Returns ``(table, lens, state, shares, source, target)``: the new table, lengths, state and counts, and for every row the page to be
    copied and the fresh one it is copied to, or -1 (int32, for ``pagedCopy`` in every layer's cache).  A refused step changes
    nothing and returns what came in; its verdict adds 32 (an origin that is no row) and 64 (a count below 0, a row's page that
    is not in the cache, a page that loses more holders than ``shares`` says it has) to those of ``pagedResize``; counts that are too
    low and are not found so are the caller's mistake.  A row that shares pages may grow by ``pagedResize`` and shrink by it as far as
    pages that it holds alone; it ends here, with origin -1.  Up to 8192 rows.
    """
    return tuple(blockAttention.pagedFork(table, free, state, shares, lens, origin, int(pageSize)))


def pagedCopy(kCache: torch.Tensor, vCache: torch.Tensor, source: torch.Tensor, target: torch.Tensor) -> None:
    """Pages ``source[i]`` of both caches into pages ``target[i]`` (int32), in place; entries below 0 are skipped.

    No page may be a target twice, or a target and a source.
    """
    blockAttention.pagedCopy(kCache, vCache, source, target)


def set_schedule_cache(capacity: int) -> None:
    """How many schedules the operators keep for metadata tensors they have seen (default 8; 0 = off).

    A call whose metadata tensors are the same objects, unmodified (PyTorch's version counters), as in an
    earlier call reuses that call's device-side plan and skips the scheduler and its host synchronisation.
    Turn it off only if metadata tensors are rewritten through raw pointers, which PyTorch cannot see."""
    blockAttention.set_schedule_cache(int(capacity))


def schedule_cache_stats() -> dict:
    hits, misses, entries, capacity = blockAttention.schedule_cache_stats()
    return {"hits": hits, "misses": misses, "entries": entries, "capacity": capacity}
