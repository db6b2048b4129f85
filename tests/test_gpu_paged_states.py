"""pagedResize with states that no call of it has left."""
import pytest
import torch

import blockedAttention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("requests", [3, 5000])
@pytest.mark.parametrize("state,verdict", [
    ([2 ** 63 - 1, 0], 16), ([2 ** 63 - 3, 0], 16), ([-2 ** 63, 0], 16), ([2 ** 32 + 2, 0], 16),      # counts that no stack holds
    ([2, 2 ** 32], 2 ** 32), ([2, -1], -1), ([2, 2 ** 40 + 1], 2 ** 40 + 1)])                         # verdicts that the operator does not know
def test_states_of_any_64_bits_are_refused_and_nothing_moves(dev, requests, state, verdict):
    """The first request gives two pages back, the second takes one, the third stays; the rest are not there."""
    table = torch.full((requests, 4), -1, dtype=torch.int32, device=dev)
    table[0, :3] = torch.tensor([5, 3, 4]); table[2, 0] = 0
    free = torch.arange(requests + 9, dtype=torch.int32, device=dev)
    lens, new = (torch.zeros(requests, dtype=torch.int64, device=dev) for _ in range(2))
    lens[:3] = torch.tensor([40, 0, 7]); new[:3] = torch.tensor([16, 5, 7])
    before = table.clone(), free.clone()
    slots, accum, after, out = blockedAttention.pagedResize(table, free, torch.tensor(state, device=dev), lens, new, 16, 8)
    assert out.tolist() == [state[0], verdict]
    assert (slots == -1).all() and (accum == 0).all() and torch.equal(after, lens)
    assert torch.equal(table, before[0]) and torch.equal(free, before[1])
