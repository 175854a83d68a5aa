"""Argument checks of tree attention, packed appends, accepted rows, forks and
compactions: every refusal comes before any CUDA call, so they run without a
GPU (the pointers are numbers that are never followed)."""
import ctypes as C

import pytest

OK, INVALID, ALIGN, WORKSPACE, UNSUPPORTED, TOO_LARGE = 0, 1, 2, 3, 5, 7


@pytest.fixture(scope="module")
def va():
    import voltattn_b200
    return voltattn_b200


def bufs(va, **kw):
    d = dict(K=4096, V=4096, scK=4096, scV=4096, q=4096, out=4096)
    d.update(kw)
    return va.VaBufs(*(d[k] for k in ("K", "V", "scK", "scV", "q", "out")))


TREE = dict(fmt=5, q_strides=None, out_strides=None, mask=4096, lens=4096, nodes=4096, table=4096, max_pages=4, B=2,
            Hq=8, Hkv=2, Q=4, page=32, pages=9, D=128, S=2, ws=4096, ws_bytes=1 << 30)


def tree(va, b=None, **kw):
    a = dict(TREE)
    a.update(kw)
    b = b or bufs(va)
    st = [None if a[k] is None else (C.c_longlong * 3)(*a[k]) for k in ("q_strides", "out_strides")]
    return va.lib().va_decode_tree(a["fmt"], C.byref(b), st[0], st[1], a["mask"], a["lens"], a["nodes"], a["table"],
                                   a["max_pages"], a["B"], a["Hq"], a["Hkv"], a["Q"], a["page"], a["pages"], a["D"],
                                   a["S"], a["ws"], a["ws_bytes"], None)


@pytest.mark.parametrize("kw,status", [
    (dict(fmt=-1), INVALID), (dict(fmt=10), INVALID),
    (dict(fmt=9), UNSUPPORTED), (dict(fmt=0), UNSUPPORTED), (dict(fmt=4), UNSUPPORTED),  # q4c+, the plain kernels' formats
    (dict(D=96), UNSUPPORTED), (dict(page=12), UNSUPPORTED), (dict(page=0), INVALID),
    (dict(mask=None), INVALID), (dict(lens=None), INVALID), (dict(table=None), INVALID),
    (dict(B=0), INVALID), (dict(Hq=7), INVALID), (dict(Hkv=0), INVALID), (dict(Q=0), INVALID), (dict(pages=0), INVALID),
    (dict(max_pages=0), INVALID), (dict(S=-1), INVALID),
    (dict(Q=65), TOO_LARGE), (dict(S=129), TOO_LARGE), (dict(max_pages=1 << 28), TOO_LARGE), (dict(B=1 << 24), TOO_LARGE),
    (dict(B=20000, S=2), TOO_LARGE),  # more row tiles than a split call has counters for
    (dict(q_strides=(4096, 1024, 132)), ALIGN), (dict(out_strides=(4096, 1028, 128)), ALIGN),
    (dict(ws=None), WORKSPACE), (dict(ws=4100), WORKSPACE), (dict(ws_bytes=100), WORKSPACE),
    (dict(S=64, ws_bytes=1 << 16), WORKSPACE)])
def test_tree_refusals(va, kw, status):
    assert tree(va, **kw) == status


@pytest.mark.parametrize("kw,status", [
    (dict(K=None), INVALID), (dict(V=None), INVALID), (dict(scK=None), INVALID), (dict(scV=None), INVALID),
    (dict(q=None), INVALID), (dict(out=None), INVALID), (dict(K=4104), ALIGN), (dict(scV=4100), ALIGN),
    (dict(q=4104), ALIGN), (dict(out=4100), ALIGN)])
def test_tree_buffer_refusals(va, kw, status):
    assert tree(va, b=bufs(va, **kw)) == status


def test_tree_workspace_and_splits(va):
    one = va.tree_workspace_bytes(2, 8, 2, 4, 128, 1)
    assert one > 0 and va.tree_workspace_bytes(2, 8, 2, 4, 128, 2) >= one + 2 * 2 * 8 * 4 * 130 * 4
    for bad in ((0, 8, 2, 4, 128, 1), (2, 7, 2, 4, 128, 1), (2, 8, 2, 65, 128, 1), (2, 8, 2, 4, 128, 129), (2, 8, 2, 4, 128, 0)):
        assert va.tree_workspace_bytes(*bad) == 0
    s = C.c_int(0)
    assert va.lib().va_suggest_tree_splits(5, 2, 7, 2, 4, 100, 128, C.byref(s)) == INVALID
    assert va.lib().va_suggest_tree_splits(9, 2, 8, 2, 4, 100, 128, C.byref(s)) == UNSUPPORTED
    assert va.lib().va_suggest_tree_splits(5, 2, 8, 2, 4, 100, 128, None) == INVALID


APPEND = dict(fmt=5, k=4096, v=4096, kind=1, ks=None, vs=None, table=4096, max_pages=4, cu=4096, pos=4096, T=5, B=2, Hkv=2,
              page=32, pages=9, D=128)


@pytest.mark.parametrize("kw,status", [
    (dict(fmt=9), UNSUPPORTED), (dict(fmt=11), INVALID), (dict(kind=3), INVALID), (dict(kind=-1), INVALID),
    (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(table=None), INVALID), (dict(cu=None), INVALID),
    (dict(pos=None), INVALID), (dict(T=-1), INVALID), (dict(B=0), INVALID), (dict(D=32), UNSUPPORTED),
    (dict(k=4104), ALIGN), (dict(ks=(260, 128)), ALIGN), (dict(vs=(256, 4)), ALIGN), (dict(kind=0, ks=(258, 128)), ALIGN),
    (dict(max_pages=1 << 28), TOO_LARGE), (dict(T=0), OK), (dict(T=0, k=None, v=None), OK)])
def test_append_refusals(va, kw, status):
    a = dict(APPEND)
    a.update(kw)
    b = bufs(va)
    st = [None if a[k] is None else (C.c_longlong * 2)(*a[k]) for k in ("ks", "vs")]
    assert va.lib().va_append_packed(a["fmt"], a["k"], a["v"], a["kind"], st[0], st[1], C.byref(b), a["table"], a["max_pages"],
                                     a["cu"], a["pos"], a["T"], a["B"], a["Hkv"], a["page"], a["pages"], a["D"], None) == status


ACCEPT = dict(fmt=5, table=4096, max_pages=4, lens=4096, nodes=4096, path=4096, accepted=4096, new=8192, B=2, P=4, Hkv=2,
              page=32, pages=9, D=128, layers=1)


@pytest.mark.parametrize("kw,status", [
    (dict(fmt=9), UNSUPPORTED), (dict(path=None), INVALID), (dict(accepted=None), INVALID), (dict(nodes=None), INVALID),
    (dict(new=None), INVALID), (dict(new=4096), INVALID), (dict(P=0), INVALID), (dict(P=65), TOO_LARGE),
    (dict(layers=0), INVALID), (dict(layers=70000), TOO_LARGE), (dict(B=70000), TOO_LARGE), (dict(D=100), UNSUPPORTED)])
def test_accept_refusals(va, kw, status):
    a = dict(ACCEPT)
    a.update(kw)
    b = bufs(va)
    assert va.lib().va_accept_tree(a["fmt"], C.byref(b), a["table"], a["max_pages"], a["lens"], a["nodes"], a["path"],
                                   a["accepted"], a["new"], a["B"], a["P"], a["Hkv"], a["page"], a["pages"], a["D"],
                                   a["layers"], None) == status


FORK = dict(fmt=5, refs=4096, table=8192, lens=12288, parent=16384, new_refs=20480, new_table=24576, new_lens=28672,
            short=32768, Bin=2, Bout=3, max_pages=4, reserve=1, Hkv=2, page=32, pages=9, D=128, layers=1, ws=4096, ws_bytes=1 << 20)


@pytest.mark.parametrize("kw,status", [
    (dict(fmt=9), UNSUPPORTED), (dict(page=12), UNSUPPORTED), (dict(refs=None), INVALID), (dict(parent=None), INVALID),
    (dict(short=None), INVALID), (dict(new_refs=4096), INVALID), (dict(new_table=8192), INVALID), (dict(new_lens=12288), INVALID),
    (dict(new_lens=16384), INVALID), (dict(reserve=-1), INVALID), (dict(Bin=0), INVALID), (dict(Bout=0), INVALID),
    (dict(Bin=4001), TOO_LARGE), (dict(Bout=4001), TOO_LARGE), (dict(ws=None), WORKSPACE), (dict(ws=4098), WORKSPACE),
    (dict(ws_bytes=8), WORKSPACE), (dict(layers=0), INVALID)])
def test_fork_refusals(va, kw, status):
    a = dict(FORK)
    a.update(kw)
    b = bufs(va)
    assert va.lib().va_fork_pages(a["fmt"], C.byref(b), a["refs"], a["table"], a["lens"], a["parent"], a["new_refs"],
                                  a["new_table"], a["new_lens"], a["short"], a["Bin"], a["Bout"], a["max_pages"], a["reserve"],
                                  a["Hkv"], a["page"], a["pages"], a["D"], a["layers"], a["ws"], a["ws_bytes"], None) == status


@pytest.mark.parametrize("kw,status", [
    (dict(fmt=9), UNSUPPORTED), (dict(page=4), UNSUPPORTED), (dict(refs=None), INVALID), (dict(used=None), INVALID),
    (dict(new_refs=4096), INVALID), (dict(new_table=8192), INVALID), (dict(ws=None), WORKSPACE), (dict(ws_bytes=64), WORKSPACE),
    (dict(layers=0), INVALID), (dict(pages=0), INVALID)])
def test_compact_refusals(va, kw, status):
    a = dict(fmt=5, refs=4096, table=8192, new_refs=20480, new_table=24576, used=32768, B=2, max_pages=4, Hkv=2, page=32,
             pages=9, D=128, layers=1, ws=4096, ws_bytes=1 << 20)
    a.update(kw)
    b = bufs(va)
    assert va.lib().va_compact_pages(a["fmt"], C.byref(b), a["refs"], a["table"], a["new_refs"], a["new_table"], a["used"],
                                     a["B"], a["max_pages"], a["Hkv"], a["page"], a["pages"], a["D"], a["layers"], a["ws"],
                                     a["ws_bytes"], None) == status


def test_python_mirror_refuses(va):
    import torch
    x = torch.zeros(4, 2, 128)
    b = va.DeviceBufs(x, x, x, x)
    with pytest.raises(ValueError):  # types
        va.append_packed("q4+", x, x.half(), b, x, 1, x, x, 1, 2, 32, 1, 128)
    with pytest.raises(ValueError):
        va.append_packed("q4+", x.int(), x.int(), b, x, 1, x, x, 1, 2, 32, 1, 128)
    with pytest.raises(ValueError):  # sizes
        va.append_packed("q4+", x, x, b, x, 1, x, x, 1, 3, 32, 1, 128)
    with pytest.raises(ValueError):  # the last dimension strided
        va.append_packed("q4+", x.expand(4, 2, 128).transpose(1, 2), x.transpose(1, 2), b, x, 1, x, x, 1, 128, 32, 1, 2)
    with pytest.raises(ValueError):
        va.decode_tree("q5", va.DeviceBufs(x, x, x, x, x, x, x), x, x, x, x, 1, 1, 1, 1, 1, 8, 1, 128)
