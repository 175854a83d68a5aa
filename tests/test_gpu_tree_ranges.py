"""bf16+ rows at the ends of fp16's range, which tree attention takes them in, and one token a sequence
against the paged single-token decode over the same cache. No reference counterpart."""
import numpy as np
import pytest

from tests import cache_ref as R
from tests.test_gpu_tree import Case, bound
from tests.test_gpu_tree_tables import Wide

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def va():
    import torch
    assert torch.cuda.is_available()
    import voltattn_b200
    return voltattn_b200


def bf16(x):
    return (np.asarray(x, np.float32).view(np.uint32) >> 16).astype(np.uint16).view(np.uint8)


def case(va, tile, L=150):
    G = {16: 4, 128: 25, 256: 50}[tile]
    c = (Case if tile == 16 else Wide)("bf16+", 1, 2 * G, 2, 5, 128, 32, [L], seed=tile)
    assert va.tree_tile_rows("bf16+", 1, 2 * G, 2, 5, c.max_pages * 32, 128) == tile
    return c


@pytest.mark.parametrize("tile", [16, 128, 256])
def test_largest_and_smallest_exact_values(va, tile):
    """bf16 has 8 bits: its values are fp16 values from 2^-17 (their last bit 2^-24) up to 65280."""
    c = case(va, tile)
    v = c.sides[1][0]
    row = np.full(128, 65280.0, np.float32)
    row[1::2] = np.float32(2.0 ** -17 * (1 + 127 / 128))
    row[3::4] *= -1
    for at in (5, 149):
        v[c.table[0, at // 32], :, at % 32] = bf16(row)
    for at in range(0, 150):  # the other rows' entries there: small ones too, so that they show
        for k in range(2):
            x = v[c.table[0, at // 32], k, at % 32].view(np.uint16)
            if at not in (5, 149):
                x[1::2] = bf16(np.full(64, 2.0 ** -16 * (1 + (at % 128) / 128), np.float32)).view(np.uint16)
    c.check(va, 2)


@pytest.mark.parametrize("tile", [16, 128, 256])
@pytest.mark.parametrize("where", ["context", "drafted"])
@pytest.mark.parametrize("S", [1, 2, 3, 4])
def test_beyond_fp16_is_infinite(va, tile, where, S):
    """65536 and more: infinite, in its dim, for the nodes that see the row; no other output changes its meaning."""
    c = case(va, tile, 400)
    j, d, v = 2, 9, c.sides[1][0]
    at = 395 - 20 if where == "context" else 400 - 5 + j
    x = v[c.table[0, at // 32], 0, at % 32].view(np.uint16)
    x[d] = bf16(np.float32([65536.0])).view(np.uint16)[0]
    want, mag = c.expect()
    got = c.run(va, S).astype(np.float64)
    G = c.Hq // 2
    for i in range(5):
        hit = np.zeros((c.Hq, 128), bool)
        hit[:G, d] = where == "context" or int(c.mask[0, i]) >> j & 1
        assert np.isposinf(got[0, i][hit]).all()
        assert (np.abs(got[0, i] - want[0, i]) <= bound(want[0, i], mag[0, i]))[~hit].all()


@pytest.mark.parametrize("fmt", R.FORMATS)
@pytest.mark.parametrize("Hq,Hkv", [(8, 8), (8, 2)])
def test_one_token_matches_the_paged_decode(va, fmt, Hq, Hkv):
    """Q = 1, no mask but its own row: the same attention as va.decode_paged, by its own kernel."""
    import torch
    B, D, page, lens = 3, 128, 64, [700, 64, 1]
    c = Case(fmt, B, Hq, Hkv, 1, D, page, lens, spare=2)
    got = c.check(va, 3)
    b = c.bufs(va)
    sc = [None if x is None else torch.nan_to_num(x, nan=0.0, posinf=0.0) for x in (b.scK, b.scV)]
    q = b.q.view(B, Hq, D)
    out = torch.empty_like(q)
    ws = torch.zeros(va.gqa_workspace_bytes(B, Hq, D, 2), dtype=torch.uint8, device="cuda")
    # (rows past the sequences' ends hold anything: clean ones for a kernel that reads whole tiles)
    rows = []
    for side, x in ((0, b.K), (1, b.V)):
        h = c.sides[side][0].copy()
        used = np.zeros((c.pages, page), bool)
        for i in range(B):
            for p in range(lens[i]):
                used[c.table[i, p // page], p % page] = True
        h[np.repeat(~used[:, None], Hkv, 1)] = 0
        rows.append(torch.from_numpy(h).cuda())
    va.decode_paged(fmt, va.DeviceBufs(rows[0], rows[1], sc[0], sc[1], q.contiguous(), out, ws), c.dev(c.table), c.max_pages, c.dev(c.lens), B, Hq,
                    Hkv, page, c.pages, D, 2)
    torch.cuda.synchronize()
    assert (np.abs(out.cpu().numpy().astype(np.float64) - got[:, 0]) <= 2e-2).all()
