"""examples/guarded_decode.py: rotation with its gradient, append and attention over a guarded 8-bit cache, run together."""
from __future__ import annotations

import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "guarded_decode.py")


@pytest.mark.parametrize("cache,tokens", [("e4m3", 48), ("int8", 48), ("e4m3", 1), ("int8", 133)])
def test_example(cache, tokens):
    spec = importlib.util.spec_from_file_location("guarded_decode", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    losses, off, bad, found = m.main(tokens, cache, quiet=True)
    assert tokens == 1 or losses[-1] < losses[0]
    # keys and values are off by half a step of their codes, 2^-4 of a value in e4m3 and 1/254 of a page's largest in int8;
    # an output is a mean of values, and the scores move it by as much again
    assert off <= (2.0 ** -4 * 2 if cache == "e4m3" else 2.0 / 127 * 2)
    assert bad == 0 and found["entries"] == [(1, 0)]
