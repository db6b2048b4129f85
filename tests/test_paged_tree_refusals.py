"""What the entry points for drafted tokens and shared pages refuse before anything reaches a GPU."""
import ctypes
import inspect

import pytest
import torch

import blockedAttention
from blockedattention_amd import capi
from test_paged_refusals import P, a_cache


def tree(parents=P, accum=P, requests=3, tokens=9, nodes=5, mask=P, depth=P):
    return capi.load().ba_paged_tree(parents, accum, requests, tokens, nodes, mask, depth, None)


def attention(cache, dtype=0, q=P, heads=4, tokens=7, table=P, table_stride=9, width=9, lens=P, accum=P, requests=3, mask=P, mask_stride=2, words=2, window=0,
              out=P, counters=P, work=None, room=0, stride=64):
    return capi.load().ba_paged_tree_attention(cache, dtype, q, stride, 256, heads, tokens, table, table_stride, width, lens, accum, requests, mask, mask_stride,
                                               words, window, 1.0, out, 64, 256, counters, work, room, None)


def keep(cache, table=P, table_stride=9, width=9, lens=P, path=P, path_stride=4, requests=3, depth=4, out=P):
    return capi.load().ba_paged_keep(cache, table, table_stride, width, lens, path, path_stride, requests, depth, out, None)


def fork(table=P, table_stride=9, width=9, free=P, pool=50, state=P, shares=P, pages=60, lens=P, origin=P, requests=3, page=16, table_out=P, out_stride=9,
         lens_out=P, state_out=P, shares_out=P, source=P, target=P, work=None, room=0):
    return capi.load().ba_paged_fork(table, table_stride, width, free, pool, state, shares, pages, lens, origin, requests, page, table_out, out_stride, lens_out,
                                     state_out, shares_out, source, target, work, room, None)


def copy(cache, source=P, target=P, copies=3):
    return capi.load().ba_paged_copy(cache, source, target, copies, None)


def test_tree_arguments():
    for bad in (dict(parents=None), dict(accum=None), dict(mask=None), dict(depth=None), dict(requests=-1), dict(tokens=-1), dict(nodes=0)):
        assert tree(**bad) == 1, bad
    for bad in (dict(nodes=1025), dict(requests=1 << 31), dict(tokens=1 << 31)):
        assert tree(**bad) == 3, bad
    assert tree(tokens=0, parents=None) == 0


@pytest.mark.parametrize("changes,status", [
    (dict(pages=-1), 1), (dict(heads=0), 1), (dict(page=0), 1), (dict(dim=0), 1), (dict(k=None), 1), (dict(v=None), 1), (dict(k_head_stride=-1), 1),
    (dict(dtype=2), 3), (dict(dtype=77), 3), (dict(dim=257), 3), (dict(page=1 << 31), 3), (dict(v_token_stride=1 << 30), 3), (dict(pages=1 << 31), 3)])
def test_caches(changes, status):
    assert attention(a_cache(**changes)) == status and keep(a_cache(**changes)) == status and copy(a_cache(**changes)) == status
    assert capi.load().ba_paged_tree_attention_workspace(a_cache(**changes), 4, 7, 3, 9) == 0


def test_attention_arguments():
    c = a_cache()
    assert attention(None) == 1
    for bad in (dict(q=None), dict(out=None), dict(counters=None), dict(lens=None), dict(accum=None), dict(table=None), dict(heads=3), dict(heads=0), dict(requests=-1),
                dict(tokens=-1), dict(width=-1), dict(window=-1), dict(table_stride=8), dict(stride=-64), dict(words=0), dict(mask_stride=1), dict(mask_stride=-2)):
        assert attention(c, **bad) == 1, bad
    assert attention(c, dtype=1) == 3 and attention(c, dtype=2) == 3
    assert attention(c, width=1 << 28, table_stride=1 << 28) == 3 and attention(c, tokens=1 << 29) == 3 and attention(c, requests=1 << 29) == 3
    assert attention(a_cache(dtype=capi.BA_F8_E4M3)) == 1                 # no scales
    assert attention(c, tokens=0) == 0
    need = capi.load().ba_paged_tree_attention_workspace(c, 4, 7, 3, 9)
    if need:
        work = dict(work=P, room=need)
        assert attention(c) == 2 and attention(c, work=P, room=need - 1) == 2 and attention(c, **dict(work, work=ctypes.c_void_p(257))) == 2


def test_keep_arguments():
    c = a_cache()
    assert keep(None) == 1
    for bad in (dict(table=None), dict(lens=None), dict(path=None), dict(out=None), dict(table_stride=8), dict(path_stride=3), dict(path_stride=-4), dict(requests=-1),
                dict(depth=-1), dict(width=-1)):
        assert keep(c, **bad) == 1, bad
    for bad in (dict(width=1 << 28, table_stride=1 << 28), dict(requests=1 << 31), dict(depth=1 << 31, path_stride=1 << 31)):
        assert keep(c, **bad) == 3, bad
    assert keep(c, requests=0) == 0


def test_fork_arguments():
    for bad in (dict(table=None), dict(free=None), dict(state=None), dict(shares=None), dict(lens=None), dict(origin=None), dict(table_out=None), dict(lens_out=None),
                dict(state_out=None), dict(shares_out=None), dict(source=None), dict(target=None), dict(requests=-1), dict(page=0), dict(width=-1), dict(pool=-1),
                dict(pages=-1), dict(table_stride=8), dict(out_stride=8)):
        assert fork(**bad) == 1, bad
    for bad in (dict(requests=8193), dict(page=1 << 30), dict(pool=1 << 31), dict(pages=1 << 31)):
        assert fork(**bad) == 3, bad
    need = capi.load().ba_paged_fork_workspace(3, 60)
    assert need > 0 and fork() == 2 and fork(work=P, room=need - 1) == 2 and fork(work=ctypes.c_void_p(128), room=need) == 2
    assert capi.load().ba_paged_fork_workspace(8193, 60) == 0 and capi.load().ba_paged_fork_workspace(3, -1) == 0


def test_copy_arguments():
    c = a_cache()
    assert copy(None) == 1
    for bad in (dict(source=None), dict(target=None), dict(copies=-1)):
        assert copy(c, **bad) == 1, bad
    assert copy(c, copies=1 << 31) == 3 and copy(a_cache(heads=1 << 19, page=1 << 10)) == 3
    assert copy(c, copies=0) == 0 and copy(a_cache(pages=0)) == 0


def test_operators_want_gpu_tensors_and_name_what_is_wrong():
    kc = torch.zeros((2, 2, 4, 8), dtype=torch.float16)
    one, two = torch.zeros(1, dtype=torch.int64), torch.zeros(2, dtype=torch.int64)
    table = torch.zeros((1, 1), dtype=torch.int32)
    for call in (lambda: blockedAttention.pagedTree(one, two, 4), lambda: blockedAttention.pagedTreeAttention(kc[0], kc, kc, table, one, two),
                 lambda: blockedAttention.pagedKeep(kc, kc, table, one, one[None]),
                 lambda: blockedAttention.pagedFork(table, table[0], two, table[0], one, one, 16), lambda: blockedAttention.pagedCopy(kc, kc, table[0], table[0])):
        with pytest.raises(RuntimeError, match="must be a GPU tensor"):
            call()


def test_signatures():
    names = lambda f: list(inspect.signature(f).parameters)  # noqa: E731
    assert names(blockedAttention.pagedTree) == ["parents", "accum", "nodes"]
    assert names(blockedAttention.pagedTreeAttention) == ["q", "kCache", "vCache", "table", "lens", "accum", "mask", "scale", "window", "kScale", "vScale"]
    assert names(blockedAttention.pagedKeep) == ["kCache", "vCache", "table", "lens", "path"]
    assert names(blockedAttention.pagedFork) == ["table", "free", "state", "shares", "lens", "origin", "pageSize"]
    assert names(blockedAttention.pagedCopy) == ["kCache", "vCache", "source", "target"]
