"""Where the entry points of the paged cache draw their limits; nothing here reaches a GPU."""
import pytest

from test_paged_refusals import a_cache, append, attention


@pytest.mark.parametrize("page,width", [(4202512, 511), (9216668, 233), (6487866, 331), (16, (1 << 27) - 1), (1, (1 << 31) - 1)])
def test_rows_of_a_table_hold_up_to_2_31_tokens(page, width):
    """width * page below 2^31 is taken, whether or not a page divides 2^31; without a workspace the call ends there."""
    for w, status in ((width, 2), (width + 1, 3)):
        assert attention(a_cache(page=page, dim=8), width=w, table_stride=w, work=None) == status


@pytest.mark.parametrize("ones", [dict(pages=1), dict(heads=1), dict(page=1), dict(pages=1, heads=1, page=1)])
def test_strides_of_dimensions_of_one_are_not_limited(ones):
    name = {"pages": "page", "heads": "head", "page": "token"}
    for stride in (0, 1 << 30, 1 << 31, (1 << 62) + 1):
        strides = {f"{array}_{name[one]}_stride": stride for array in "kv" for one in ones}
        assert append(a_cache(**ones, **strides), tokens=0) == 0
        assert attention(a_cache(**ones, **strides), heads=2, requests=0) == 0
        assert attention(a_cache(**ones, **strides), heads=2, work=None) == 2
        if stride > 1 << 40:                                              # where there are more entries they are
            assert append(a_cache(**strides), tokens=0) != 0
