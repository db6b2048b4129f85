"""A draft whose step is refused, in the order in which a program that does not wait for the verdict makes its calls: nothing of the cache changes."""
import pytest
import torch

import blockedAttention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("room", [0, 1])
def test_a_refused_draft_changes_nothing(dev, room):
    """Row 0 had pages once that row 1 has now; its table still names them.  room 1: the same with a step that is not refused."""
    page, i64 = 4, dict(dtype=torch.int64, device=dev)
    k, v = (torch.randn((7, 2, page, 16), dtype=torch.bfloat16, device=dev) for _ in range(2))
    table, free = torch.zeros((2, 6), dtype=torch.int32, device=dev), torch.arange(7, dtype=torch.int32, device=dev)
    state, lens = torch.tensor([5 + 2 * room, 0], **i64), torch.zeros(2, **i64)
    for new in ([18, 0], [3, 0], [3, 16]):                    # five pages, one; four of them are row 1's then
        _, _, lens, state = blockedAttention.pagedResize(table, free, state, lens, torch.tensor(new, **i64), page, 18)
    assert state.tolist() == [2 * room, 0] and table[0, 1:5].tolist() == sorted(table[1, :4].tolist(), reverse=table[0, 1] > table[0, 2])
    before = [t.clone() for t in (k, v, table, free, lens)]
    new = lens + torch.tensor([6, 0], **i64)
    slots, accum, grown, state = blockedAttention.pagedResize(table, free, state, lens, new, page, 6)
    assert (state[1].item() == 0) == bool(room)
    x = torch.ones((2, 6, 16), dtype=torch.bfloat16, device=dev) * torch.arange(6, device=dev)[None, :, None]
    blockedAttention.pagedAppend(x, x, k, v, slots)
    path = torch.where(state[1] == 0, torch.tensor([[1, 3, 5], [-1, -1, -1]], **i64), -1)
    kept = blockedAttention.pagedKeep(k, v, table, lens, path)
    assert kept.tolist() == [6 if room else 3, 16]
    if room:
        for c in (k, v):
            assert [c[int(table[0, t // page]), 0, t % page, 0].item() for t in (3, 4, 5)] == [1, 3, 5]
    else:
        assert all(torch.equal(a, b) for a, b in zip(before, (k, v, table, free, grown)))
