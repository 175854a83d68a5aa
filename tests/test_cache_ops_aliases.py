"""Outputs of accepted rows, forks and compactions that lie in their inputs or in one another:
other CTAs still read what one has written already, so they are refused. Before any CUDA call, so
without a GPU (the pointers are numbers that are never followed)."""
import ctypes as C

import pytest

from tests.test_cache_ops_refusals import ACCEPT, FORK, INVALID, WORKSPACE, bufs

# 4-byte elements at B = 2, max_pages = 4, P = 4, 9 pages; what is not named lies elsewhere
ACCEPT_AT = dict(table=0x10000, lens=0x11000, nodes=0x12000, path=0x13000, accepted=0x14000, new=0x15000)
PAGES_AT = dict(refs=0x10000, table=0x11000, lens=0x12000, parent=0x13000, new_refs=0x14000, new_table=0x15000, new_lens=0x16000,
                short=0x17000, ws=0x18000, ws_bytes=1024)


@pytest.fixture(scope="module")
def va():
    import voltattn_b200
    return voltattn_b200


def accept(va, **kw):
    a = dict(ACCEPT)
    a.update(ACCEPT_AT)
    a.update(kw)
    b = bufs(va)
    return va.lib().va_accept_tree(a["fmt"], C.byref(b), a["table"], a["max_pages"], a["lens"], a["nodes"], a["path"],
                                   a["accepted"], a["new"], a["B"], a["P"], a["Hkv"], a["page"], a["pages"], a["D"],
                                   a["layers"], None)


def fork(va, **kw):
    a = dict(FORK)
    a.update(PAGES_AT)
    a.update(kw)
    b = bufs(va)
    return va.lib().va_fork_pages(a["fmt"], C.byref(b), a["refs"], a["table"], a["lens"], a["parent"], a["new_refs"],
                                  a["new_table"], a["new_lens"], a["short"], a["Bin"], a["Bout"], a["max_pages"], a["reserve"],
                                  a["Hkv"], a["page"], a["pages"], a["D"], a["layers"], a["ws"], a["ws_bytes"], None)


def compact(va, **kw):
    a = dict(fmt=5, B=2, max_pages=4, Hkv=2, page=32, pages=9, D=128, layers=1, **PAGES_AT)
    a.update(kw)
    b = bufs(va)
    return va.lib().va_compact_pages(a["fmt"], C.byref(b), a["refs"], a["table"], a["new_refs"], a["new_table"], a["short"],
                                     a["B"], a["max_pages"], a["Hkv"], a["page"], a["pages"], a["D"], a["layers"], a["ws"],
                                     a["ws_bytes"], None)


@pytest.mark.parametrize("what,last", [("table", 8), ("lens", 2), ("nodes", 2), ("path", 8), ("accepted", 2)])
def test_accept(va, what, last):
    at = ACCEPT_AT[what]
    for new in (at, at - 4, at + 4 * (last - 1)):
        assert accept(va, new=new) == INVALID


@pytest.mark.parametrize("out,size", [("new_refs", 9), ("new_table", 12), ("new_lens", 3), ("short", 1)])
def test_fork(va, out, size):
    sizes = dict(refs=9, table=8, lens=2, parent=3, new_refs=9, new_table=12, new_lens=3, short=1, ws=18)
    for other, n in sizes.items():
        if other == out:
            continue
        at = PAGES_AT[other]
        for p in (at, at - 4 * (size - 1), at + 4 * (n - 1)):
            assert fork(va, **{out: p}) == INVALID, other
        if other != "ws":  # next to it (the missing workspace is refused after that)
            assert fork(va, ws=None, **{out: at - 4 * size}) == WORKSPACE, other


@pytest.mark.parametrize("out,size", [("new_refs", 9), ("new_table", 8), ("short", 1)])
def test_compact(va, out, size):
    sizes = dict(refs=9, table=8, new_refs=9, new_table=8, short=1, ws=28)
    for other, n in sizes.items():
        if other == out:
            continue
        at = PAGES_AT[other]
        for p in (at, at - 4 * (size - 1), at + 4 * (n - 1)):
            assert compact(va, **{out: p}) == INVALID, other
        if other != "ws":
            assert compact(va, ws=None, **{out: at - 4 * size}) == WORKSPACE, other
