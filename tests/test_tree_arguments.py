"""What the Python mirror of the cache operators takes: q and out of the right type and shape (a
tensor of another layout would be read with the wrong strides), integer arrays of int32. Refusals come
before any CUDA call; no GPU needed for them."""
import types

import pytest
import torch

B, Hq, Hkv, Q, D = 2, 8, 2, 3, 128


@pytest.fixture(scope="module")
def va():
    import voltattn_b200
    return voltattn_b200


def call(va, **kw):
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    a = dict(q=torch.zeros(B, Q, Hq, D, dtype=torch.float16), out=torch.zeros(B, Q, Hq, D, dtype=torch.float16),
             mask=torch.zeros(B, Q, dtype=torch.int64), lens=i32(B), nodes=i32(B), table=i32(B, 4))
    a.update(kw)
    x = torch.zeros(64, dtype=torch.uint8)
    # (no workspace: a call whose arguments pass is refused for that, before any CUDA call)
    b = va.DeviceBufs(x, x, x, x, a["q"], a["out"], None)
    va.decode_tree("q4+", b, a["mask"], a["lens"], a["nodes"], a["table"], 4, B, Hq, Hkv, Q, 32, 1, D,
                   stream=types.SimpleNamespace(cuda_stream=None))


def taken(va, **kw):
    with pytest.raises(va.VoltAttnError):
        call(va, **kw)


H = torch.float16


@pytest.mark.parametrize("bad", [
    dict(q=torch.zeros(B, Q, Hq, D, dtype=torch.bfloat16)), dict(q=torch.zeros(B, Q, Hq, D)),
    dict(out=torch.zeros(B, Q, Hq, D, dtype=torch.bfloat16)), dict(out=torch.zeros(B, Q, Hq, D)),
    dict(q=torch.zeros(B, Hq, Q, D, dtype=H)), dict(out=torch.zeros(B, Hq, Q, D, dtype=H)),  # another order
    dict(q=torch.zeros(B, Q - 1, Hq, D, dtype=H)), dict(q=torch.zeros(B - 1, Q, Hq, D, dtype=H)),  # too small
    dict(q=torch.zeros(B, Q, Hq, D + 8, dtype=H)), dict(q=torch.zeros(B * Q * Hq * D - 1, dtype=H)),
    dict(q=torch.zeros(B * (Q + 1), Hq, D, dtype=H)),  # flat, and not of this size
    dict(out=torch.zeros(B, Q, Hq, 2 * D, dtype=H)[..., ::2]), dict(out=torch.zeros(Hq, B * Q, D, dtype=H).transpose(0, 1)),
    dict(mask=torch.zeros(B, Q, dtype=torch.int32)), dict(mask=torch.zeros(B, Q, dtype=torch.bool)),
    dict(mask=torch.zeros(Q, B, dtype=torch.int64).T), dict(mask=torch.zeros(1, Q, dtype=torch.int64).expand(B, Q)),
    dict(mask=torch.zeros(B, Q - 1, dtype=torch.int64)), dict(mask=torch.zeros(B, Q + 1, dtype=torch.int64)),
    dict(lens=torch.zeros(B, dtype=torch.int64)), dict(nodes=torch.zeros(B, dtype=torch.int64)),
    dict(lens=torch.zeros(B)), dict(lens=torch.zeros(2 * B, dtype=torch.int32)[::2]), dict(lens=torch.zeros(B - 1, dtype=torch.int32)),
    dict(table=torch.zeros(B, 4, dtype=torch.int64)), dict(table=torch.zeros(B, 8, dtype=torch.int32)[:, :4]),
    dict(table=torch.zeros(B, 3, dtype=torch.int32)), dict(table=torch.zeros(B, 5, dtype=torch.int32))],
    ids=lambda d: "-".join(f"{k}{tuple(v.shape)}{str(v.dtype)[6:]}" for k, v in d.items()))
def test_decode_tree_refuses(va, bad):
    with pytest.raises(ValueError):
        call(va, **bad)


@pytest.mark.parametrize("good", [
    dict(), dict(nodes=None), dict(q=torch.zeros(B * Q * Hq * D, dtype=H)), dict(q=torch.zeros(B * Q, Hq, D, dtype=H)),
    dict(q=torch.zeros(B, Q, Hq + 4, D, dtype=H)[:, :, 2:2 + Hq]), dict(out=torch.zeros(B, Hq, Q, D, dtype=H).transpose(1, 2)),
    dict(q=torch.zeros(B, Q + 2, Hq, D, dtype=H)), dict(q=torch.zeros(B + 1, Q, Hq, D, dtype=H)),
    dict(mask=torch.zeros(B, Q, dtype=torch.uint64)), dict(mask=torch.zeros(B * Q, dtype=torch.int64)),
    dict(mask=torch.zeros(B + 2, Q, dtype=torch.int64)), dict(lens=torch.zeros(B + 3, dtype=torch.int32)),
    dict(table=torch.zeros(B + 1, 4, dtype=torch.int32)), dict(table=torch.zeros(B * 4, dtype=torch.int32))],
    ids=lambda d: "-".join(d) or "plain")
def test_decode_tree_takes(va, good):
    taken(va, **good)


def test_width_of_one(va):
    """One node a sequence, one page a table: wider arrays are still not taken for them."""
    one = lambda w, t: torch.zeros(B, w, dtype=t)  # noqa: E731
    x, s = torch.zeros(64, dtype=torch.uint8), types.SimpleNamespace(cuda_stream=None)
    rows = torch.zeros(B, 1, Hq, D, dtype=H)
    b, n = va.DeviceBufs(x, x, x, x, rows, rows, None), torch.zeros(B, dtype=torch.int32)
    for w, v in ((4, 1), (1, 4)):
        with pytest.raises(ValueError):
            va.decode_tree("q4+", b, one(w, torch.int64), n, n, one(v, torch.int32), 1, B, Hq, Hkv, 1, 32, 1, D, stream=s)
    with pytest.raises(va.VoltAttnError):
        va.decode_tree("q4+", b, one(1, torch.int64), n, n, one(1, torch.int32), 1, B, Hq, Hkv, 1, 32, 1, D, stream=s)


@pytest.mark.gpu
@pytest.mark.parametrize("more", [(0, 0), (0, 5), (2, 0), (1, 3)])
def test_contiguous_q_and_out_of_more_nodes(va, more):
    """The first B sequences and Q nodes of larger contiguous tensors."""
    import numpy as np
    from tests.test_gpu_tree import Case, bound
    c = Case("q4+", 3, 8, 2, 5, 128, 32, [100, 41, 260])
    want, mag = c.expect()
    b = c.bufs(va)
    q = torch.full((3 + more[0], 5 + more[1], 8, 128), float("nan"), dtype=H, device="cuda")
    out = torch.full(q.shape, 7.0, dtype=H, device="cuda")
    q[:3, :5] = b.q
    b.q, b.out = q, out
    va.decode_tree(c.fmt, b, *c.args(), S=2)
    got = out.cpu().numpy().astype(np.float64)
    assert (np.abs(got[:3, :5] - want) <= bound(want, mag)).all()
    got[:3, :5] = 7.0
    assert (got == 7.0).all()
