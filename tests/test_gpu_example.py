"""The speculative-decoding example end to end: trees give the tokens of
one-by-one decoding, in fewer steps. No reference counterpart."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu


def test_tree_speculation_example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "tree_speculation.py")
    spec = importlib.util.spec_from_file_location("tree_speculation", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    one, tree = m.main(["--tokens", "20"])
    assert tree < one
