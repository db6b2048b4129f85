"""Where the entry points of the paged cache draw their limits; nothing here reaches a GPU."""
import pytest

from test_paged_refusals import a_cache, attention


@pytest.mark.parametrize("page,width", [(4202512, 511), (9216668, 233), (6487866, 331), (16, (1 << 27) - 1), (1, (1 << 31) - 1)])
def test_rows_of_a_table_hold_up_to_2_31_tokens(page, width):
    """width * page below 2^31 is taken, whether or not a page divides 2^31; without a workspace the call ends there."""
    for w, status in ((width, 2), (width + 1, 3)):
        assert attention(a_cache(page=page, dim=8), width=w, table_stride=w, work=None) == status
