"""What the entry points of the paged cache refuse before anything reaches a GPU."""
import ctypes
import inspect

import pytest
import torch

import blockedAttention
from blockedattention_amd import capi


def a_cache(**changes):
    c = capi.PagedCache(256, 256, None, None, 4, 2, 16, 64, 2048, 1024, 64, 2048, 1024, 64, capi.BA_F16)
    for name, value in changes.items():
        setattr(c, name, value)
    return ctypes.byref(c)


P = ctypes.c_void_p(256)          # an address that nothing reads


def attention(cache, dtype=0, q=P, heads=4, requests=3, table=P, table_stride=9, width=9, lens=P, window=0, out=P, counters=P, work=P, room=1 << 30, stride=64):
    return capi.load().ba_paged_attention(cache, dtype, q, stride, 256, heads, requests, table, table_stride, width, lens, window, 1.0, out, 64, 256,
                                          counters, work, room, None)


def append(cache, dtype=0, k=P, v=P, slots=P, tokens=5, stride=64):
    return capi.load().ba_paged_append(cache, dtype, k, stride, 128, v, 64, 128, slots, tokens, None)


@pytest.mark.parametrize("changes,status", [
    (dict(pages=-1), 1), (dict(heads=0), 1), (dict(page=0), 1), (dict(dim=0), 1), (dict(k=None), 1), (dict(v=None), 1), (dict(k_head_stride=-1), 1),
    (dict(k_scale=256), 1), (dict(dtype=9), 1), (dict(dtype=2), 3), (dict(dtype=77), 3), (dict(dim=257), 3), (dict(page=1 << 31), 3),
    (dict(v_token_stride=1 << 30), 3), (dict(pages=1 << 31), 3)])
def test_caches(changes, status):
    assert attention(a_cache(**changes)) == status
    assert append(a_cache(**changes)) == status
    assert capi.load().ba_paged_attention_workspace(a_cache(**changes), 4, 3, 9) == 0


def test_attention_arguments():
    c = a_cache()
    assert attention(None) == 1
    for bad in (dict(q=None), dict(out=None), dict(counters=None), dict(lens=None), dict(table=None), dict(heads=3), dict(heads=0), dict(requests=-1), dict(width=-1),
                dict(window=-1), dict(table_stride=8), dict(stride=-64)):
        assert attention(c, **bad) == 1, bad
    assert attention(c, dtype=1) == 3 and attention(c, dtype=2) == 3
    assert attention(c, width=1 << 28, table_stride=1 << 28) == 3         # more than 2^31 tokens a row
    assert attention(c, requests=0) == 0
    need = capi.load().ba_paged_attention_workspace(c, 4, 3, 9)
    if need:
        assert attention(c, room=need - 1) == 2 and attention(c, work=None) == 2 and attention(c, work=ctypes.c_void_p(257)) == 2


def test_append_arguments():
    c = a_cache()
    assert append(None) == 1
    for bad in (dict(k=None), dict(v=None), dict(slots=None), dict(tokens=-1), dict(stride=-1)):
        assert append(c, **bad) == 1, bad
    assert append(c, dtype=1) == 3 and append(c, dtype=2) == 3 and append(c, tokens=1 << 31) == 3
    assert append(a_cache(pages=1 << 30), dtype=0) == 3                   # places past 2^31
    assert append(c, tokens=0) == 0 and append(a_cache(pages=0)) == 0


def test_resize_arguments():
    def resize(table=P, table_stride=9, width=9, free=P, pool=50, state=P, lens=P, new=P, requests=3, page=16, slots=P, tokens=7, accum=P, out=P, state_out=P):
        return capi.load().ba_paged_resize(table, table_stride, width, free, pool, state, lens, new, requests, page, slots, tokens, accum, out, state_out,
                                           None, 0, None)
    for bad in (dict(table=None), dict(free=None), dict(state=None), dict(lens=None), dict(new=None), dict(slots=None), dict(accum=None), dict(out=None),
                dict(state_out=None), dict(requests=-1), dict(page=0), dict(width=-1), dict(tokens=-1), dict(pool=-1), dict(table_stride=8)):
        assert resize(**bad) == 1, bad
    for bad in (dict(tokens=1 << 31), dict(page=1 << 30), dict(requests=1 << 29), dict(pool=1 << 31)):
        assert resize(**bad) == 3, bad


def test_operators_want_gpu_tensors_and_name_what_is_wrong():
    kc = torch.zeros((2, 2, 4, 8), dtype=torch.float16)
    one = torch.zeros(1, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="must be a GPU tensor"):
        blockedAttention.pagedAttention(torch.zeros((2, 1, 8)), kc, kc, torch.zeros((1, 1), dtype=torch.int32), one)
    with pytest.raises(RuntimeError, match="must be a GPU tensor"):
        blockedAttention.pagedAppend(torch.zeros((2, 1, 8)), torch.zeros((2, 1, 8)), kc, kc, one)
    with pytest.raises(RuntimeError, match="must be a GPU tensor"):
        blockedAttention.pagedResize(torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int64), one, one, 16, 1)


def test_signatures():
    names = lambda f: list(inspect.signature(f).parameters)  # noqa: E731
    assert names(blockedAttention.pagedResize) == ["table", "free", "state", "lens", "newLens", "pageSize", "tokens"]
    assert names(blockedAttention.pagedAppend) == ["k", "v", "kCache", "vCache", "slots", "kScale", "vScale"]
    assert names(blockedAttention.pagedAttention) == ["q", "kCache", "vCache", "table", "lens", "scale", "window", "kScale", "vScale"]
