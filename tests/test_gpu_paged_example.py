"""The paged cache's operators as a program uses them together: examples/paged_answers.py.

Values have about unit variance and attention averages them, so results stay below 5 in size: one rounding to bf16 is at most
2^-8 of that, one of each probability (2^-8 of sum p |v|, below 5 too) as much again.
"""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", ["bf16", "fp8"])
def test_answers_match_dense_attention(dev, cache):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_answers.py")
    spec = importlib.util.spec_from_file_location("paged_answers", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    worst, answered = example.main(cache, steps=60, seed=1)
    assert answered > 100 and worst <= 2 * 5 * 2.0 ** -8
