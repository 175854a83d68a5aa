"""The speculative-decoding example with prompts of one token, which leave nothing to prefill. No
reference counterpart."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("prompts", [[[3]], [[3], [5, 6, 7]], [[9], [4]]])
def test_prompts_of_one_token(prompts):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "tree_speculation.py")
    spec = importlib.util.spec_from_file_location("tree_speculation", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    model = m.ToyModel("cuda:0")
    plain, one, _ = m.decode(model, prompts, 6, "cuda:0")
    tree, steps, _ = m.decode(model, prompts, 6, "cuda:0", drafts=plain)
    assert tree == plain and steps <= one
