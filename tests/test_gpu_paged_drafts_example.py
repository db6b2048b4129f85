"""The operators of drafted and branching answers as a program uses them together: examples/paged_drafts.py.

Values stay below 6 in size (variance about 1.25, 10^5 of them) and attention averages them: one rounding to bf16 is at most 2^-8 of that, one of each
probability, and of the sum that they are divided by, 2^-8 of sum p |v| (below 6 too) as much again.
"""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", ["bf16", "fp8"])
def test_drafts_match_dense_attention(dev, cache):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_drafts.py")
    spec = importlib.util.spec_from_file_location("paged_drafts", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    worst, answered, forked = example.main(cache, steps=30, seed=2)
    assert answered > 1000 and forked >= 10 and worst <= 3 * 6 * 2.0 ** -8
