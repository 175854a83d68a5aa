"""Masks and integer arrays that are not aligned to their elements (a load there would fault) are
refused, before any CUDA call, so without a GPU (the pointers are numbers that are never followed)."""
import ctypes as C

import pytest

from tests import test_cache_ops_aliases as AL
from tests import test_cache_ops_refusals as A


@pytest.fixture(scope="module")
def va():
    import voltattn_b200
    return voltattn_b200


@pytest.mark.parametrize("what,by", [("mask", 4), ("mask", 1), ("lens", 2), ("nodes", 2), ("table", 1)])
def test_tree(va, what, by):
    assert A.tree(va, **{what: 4096 + by}) == A.ALIGN


@pytest.mark.parametrize("what", ["table", "cu", "pos"])
def test_append(va, what):
    a = dict(A.APPEND)
    a[what] += 2
    b = A.bufs(va)
    assert va.lib().va_append_packed(a["fmt"], a["k"], a["v"], a["kind"], None, None, C.byref(b), a["table"], a["max_pages"],
                                     a["cu"], a["pos"], a["T"], a["B"], a["Hkv"], a["page"], a["pages"], a["D"], None) == A.ALIGN


@pytest.mark.parametrize("what", list(AL.ACCEPT_AT))
def test_accept(va, what):
    assert AL.accept(va, **{what: AL.ACCEPT_AT[what] + 2}) == A.ALIGN


@pytest.mark.parametrize("what", [k for k in AL.PAGES_AT if k not in ("ws", "ws_bytes")])
def test_fork(va, what):
    assert AL.fork(va, **{what: AL.PAGES_AT[what] + 2}) == A.ALIGN


@pytest.mark.parametrize("what", ["refs", "table", "new_refs", "new_table", "short"])
def test_compact(va, what):
    assert AL.compact(va, **{what: AL.PAGES_AT[what] + 2}) == A.ALIGN
