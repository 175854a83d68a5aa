"""Types and shapes of the arrays that the Python mirror of the append, accept, fork and compact
operators takes: an int64 array (a cumsum, say) would be read as int32 pairs. Refusals come before any
CUDA call; no GPU needed."""
import types

import pytest
import torch

B, Hkv, D, PAGE, PAGES, MP, P = 3, 2, 128, 32, 9, 4, 5
STREAM = types.SimpleNamespace(cuda_stream=None)


@pytest.fixture(scope="module")
def va():
    import voltattn_b200
    return voltattn_b200


def ints(*s):
    return torch.zeros(*s, dtype=torch.int32)


def pool(va):
    # (no K: a call whose arguments pass is refused for that, before any CUDA call)
    x = torch.zeros(64, dtype=torch.uint8)
    return va.DeviceBufs(None, x, x, x)


def append(va, **kw):
    a = dict(k=torch.zeros(7, Hkv, D), v=torch.zeros(7, Hkv, D), table=ints(B, MP), cu=ints(B + 1), pos=ints(B))
    a.update(kw)
    va.append_packed("q4+", a["k"], a["v"], pool(va), a["table"], MP, a["cu"], a["pos"], B, Hkv, PAGE, PAGES, D, stream=STREAM)


def accept(va, **kw):
    a = dict(table=ints(B, MP), lens=ints(B), nodes=ints(B), path=ints(B, P), accepted=ints(B), new=ints(B))
    a.update(kw)
    va.accept_tree("q4+", pool(va), a["table"], MP, a["lens"], a["nodes"], a["path"], a["accepted"], a["new"], B, P, Hkv, PAGE, PAGES, D,
                   stream=STREAM)


def fork(va, **kw):
    a = dict(refs=ints(PAGES), table=ints(B, MP), lens=ints(B), parent=ints(B + 2), new_refs=ints(PAGES), new_table=ints(B + 2, MP),
             new_lens=ints(B + 2), short=ints(1))
    a.update(kw)
    va.fork_pages("q4+", pool(va), a["refs"], a["table"], a["lens"], a["parent"], a["new_refs"], a["new_table"], a["new_lens"], a["short"],
                  B, B + 2, MP, 1, Hkv, PAGE, PAGES, D, stream=STREAM)


def compact(va, **kw):
    a = dict(refs=ints(PAGES), table=ints(B, MP), new_refs=ints(PAGES), new_table=ints(B, MP), used=ints(1))
    a.update(kw)
    va.compact_pages("q4+", pool(va), a["refs"], a["table"], a["new_refs"], a["new_table"], a["used"], B, MP, Hkv, PAGE, PAGES, D,
                     stream=STREAM)


SIZES = {append: dict(table=(B, MP), cu=(B + 1,), pos=(B,)),
         accept: dict(table=(B, MP), lens=(B,), nodes=(B,), path=(B, P), accepted=(B,), new=(B,)),
         fork: dict(refs=(PAGES,), table=(B, MP), lens=(B,), parent=(B + 2,), new_refs=(PAGES,), new_table=(B + 2, MP),
                    new_lens=(B + 2,), short=(1,)),
         compact: dict(refs=(PAGES,), table=(B, MP), new_refs=(PAGES,), new_table=(B, MP), used=(1,))}
EACH = [(f, name, shape) for f, names in SIZES.items() for name, shape in names.items()]


@pytest.mark.parametrize("f,name,shape", EACH, ids=lambda x: x if isinstance(x, str) else getattr(x, "__name__", ""))
def test_arrays(va, f, name, shape):
    front = (shape[0] + 2, *shape[1:])
    bad = [torch.zeros(shape, dtype=torch.int64), torch.zeros(shape), ints(*shape).flatten()[1:], ints(2 * shape[0], *shape[1:])[::2]]
    if shape == (1,):
        bad.pop()
    if len(shape) == 2:
        bad += [ints(shape[0], shape[1] + 1), ints(shape[0], shape[1] + 1)[:, :shape[1]], ints(shape[1], shape[0]).T]
    for t in bad:
        with pytest.raises(ValueError):
            f(va, **{name: t})
    for t in (ints(*shape), ints(*front), ints(*shape).flatten()):
        with pytest.raises(va.VoltAttnError):
            f(va, **{name: t})


def test_rows_of_another_layout(va):
    for shape in ((7, 2 * Hkv, D // 2), (7, Hkv // 2, 2 * D), (7, D, Hkv)):
        x = torch.zeros(shape)
        with pytest.raises(ValueError):
            append(va, k=x, v=x)
    for x in (torch.zeros(7, Hkv, D), torch.zeros(7, 3 * Hkv, D)[:, Hkv:2 * Hkv], torch.zeros(7 * Hkv * D), torch.zeros(7, Hkv * D)):
        with pytest.raises(va.VoltAttnError):
            append(va, k=x, v=x)
