"""The serving loop of examples/paged_serving.py: requests join and leave, chunks
run beside single tokens, pages are reused."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                    "paged_serving.py")


@pytest.mark.parametrize("pages", ["same", "int8", "e4m3"])
def test_serving_loop(sm100, pages):
    spec = importlib.util.spec_from_file_location("paged_serving", PATH)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    drawn, worst = example.serve(pages, steps=60, verbose=False)
    assert sorted(len(d) for d in drawn) == [4, 8, 12, 20, 30]
    # values of a few units (projections of unit-variance rows): bf16 results, and bf16 keys
    # read back against the cache's own, differ by a few roundings of 2^-8
    assert worst <= 0.06
