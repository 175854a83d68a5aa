"""Tree attention in the tiles of 128 and 256 query rows: strides, streams and graphs, far pages, sizes
of scales, default nodes, and one workspace for both kernels. Every case asserts the tile that it runs in.
No reference counterpart."""
import numpy as np
import pytest

from tests import cache_ref as R
from tests.test_gpu_tree import Case, bound
from tests.test_gpu_tree_tables import Wide

pytestmark = pytest.mark.gpu
TILES = [(128, 128), (256, 128), (128, 64)]


@pytest.fixture(scope="module")
def va():
    import torch
    assert torch.cuda.is_available()
    import voltattn_b200
    return voltattn_b200


def large(va, fmt, B, G, Hkv, Q, D, page, lens, tile, **kw):
    c = Wide(fmt, B, G * Hkv, Hkv, Q, D, page, lens, **kw)
    assert va.tree_tile_rows(fmt, B, G * Hkv, Hkv, Q, c.max_pages * page, D) == tile
    return c


def heads(tile):
    return 25 if tile == 128 else 50  # of five nodes: 125 or 250 query rows


@pytest.mark.parametrize("fmt", R.FORMATS)
@pytest.mark.parametrize("tile,D", TILES)
def test_strides_streams_and_graphs(va, fmt, tile, D):
    """q as a slice of a fused projection, out with another order of dimensions, on the caller's stream, in a graph."""
    import torch
    G, Hkv, Q = heads(tile), 2, 5
    c = large(va, fmt, 2, G, Hkv, Q, D, 32, [200, 333], tile)
    want, mag = c.expect()
    b = c.bufs(va, 3)
    H = G * Hkv
    fused = torch.full((2, Q, H + 4, D), float("nan"), dtype=torch.float16, device="cuda")
    fused[:, :, 2:2 + H] = b.q
    b.q = fused[:, :, 2:2 + H]
    store = torch.full((2, H, Q, D + 8), float("nan"), dtype=torch.float16, device="cuda")
    b.out = store[..., :D].transpose(1, 2)
    a = c.args()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        va.decode_tree(c.fmt, b, *a, S=3)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            va.decode_tree(c.fmt, b, *a, S=3)
        store.fill_(float("nan"))
        g.replay()
    torch.cuda.synchronize()
    assert (np.abs(b.out.cpu().numpy() - want) <= bound(want, mag)).all()
    assert torch.isnan(store[..., D:]).all()


@pytest.mark.parametrize("fmt", ["f16+", "q8+"])
def test_offsets_past_32_bits(va, fmt):
    """Pages behind the first 4 GiB of each buffer of rows: tensor copies (f16+) and bulk copies."""
    import torch
    G, Hkv, Q, page = 25, 2, 5, 64
    c = large(va, fmt, 1, G, Hkv, Q, 128, page, [100], 128, spare=0)
    per = Hkv * page * R.row_bytes(fmt, 128)
    pages = (9 << 29) // per
    lo = pages - c.pages
    b = c.bufs(va, 2)
    for name, size in (("K", per), ("V", per), ("scK", Hkv * page * 4), ("scV", Hkv * page * 4)):
        src = getattr(b, name)
        if src is None:
            continue
        src = src.reshape(-1).view(torch.uint8)
        big = torch.zeros(pages * size, dtype=torch.uint8, device="cuda")
        big[lo * size:] = src
        setattr(b, name, big)
    a = list(c.args())
    a[3] = torch.where(a[3] >= 0, a[3] + lo, a[3])
    a[10] = pages
    va.decode_tree(c.fmt, b, *a, S=2)
    want, mag = c.expect()
    assert (np.abs(b.out.cpu().numpy().astype(np.float64) - want) <= bound(want, mag)).all()


@pytest.mark.parametrize("tile,D", TILES)
@pytest.mark.parametrize("fmt,spread", [("q8+", 3e-4), ("q8+", 2000.0), ("q4+", 1e-3), ("q4+", 8000.0), ("q3+", 5000.0), ("f8+", 4000.0),
                                        ("f16+", 2e-3), ("bf16+", 1e-2)])
def test_scales_of_any_size(va, fmt, spread, tile, D):
    c = large(va, fmt, 1, heads(tile), 2, 5, D, 32, [400], tile, spread=spread)
    c.q[:] = (c.q.astype(np.float32) / max(1.0, spread)).astype(np.float16)
    c.check(va, 2)


@pytest.mark.parametrize("fmt", ["q4+", "f16+"])
@pytest.mark.parametrize("tile,D", TILES)
def test_nodes_default(va, fmt, tile, D):
    c = large(va, fmt, 2, heads(tile), 2, 5, D, 32, [50, 90], tile)
    b = c.bufs(va)
    a = list(c.args())
    a[2] = None
    va.decode_tree(c.fmt, b, *a, S=2)
    want, mag = c.expect()
    assert (np.abs(b.out.cpu().numpy() - want) <= bound(want, mag)).all()


@pytest.mark.parametrize("fmt", ["q4+", "f16+", "q3+", "f8+", "bf16+"])
@pytest.mark.parametrize("tile", [128, 256])
def test_one_workspace_for_both_kernels(va, fmt, tile):
    """Calls of large and small tiles in turn over one workspace; any number of splits, and the same bits again."""
    import torch
    c = large(va, fmt, 2, heads(tile), 2, 5, 128, 64, [2100, 900], tile)
    small = Case(fmt, 7, 8, 8, 2, 64, 8, [300, 2, 9, 100, 5, 40, 1])
    assert va.tree_tile_rows(fmt, 7, 8, 8, 2, small.max_pages * 8, 64) == 16
    ws = torch.zeros(va.tree_workspace_bytes(2, 100, 2, 64, 128, 32), dtype=torch.uint8, device="cuda")
    for S in (1, 2, 5, 17, 0):
        first = c.check(va, S, ws)
        small.check(va, 3, ws)
        assert (c.run(va, S, ws).astype(np.float64) == first).all()
        assert not ws[:65536].any()  # the counters, as every call leaves them


@pytest.mark.parametrize("fmt", ["f16+", "bf16+", "f8+", "q4+"])
@pytest.mark.parametrize("what", ["nan", "inf", "-inf"])
@pytest.mark.parametrize("tile", [128, 256])
def test_unseen_rows(va, fmt, what, tile):
    """A drafted row of inf or nan reaches the nodes that see it only; the others keep their bits."""
    Q, j = 5, 2
    c = large(va, fmt, 2, heads(tile), 2, Q, 128, 32, [150, Q], tile, seed=tile)
    clean = c.run(va, 2)
    bad = float(what)
    for b in range(2):
        r = int(c.lens[b]) - Q + j
        for codes, scales in c.sides:
            at = (c.table[b, r // 32], slice(None), r % 32)
            if scales is not None:
                scales[at] = bad
            elif fmt == "f16+":
                codes[at] = np.full(128, bad, np.float16).view(np.uint8)
            else:
                codes[at] = (np.full(128, bad, np.float32).view(np.uint32) >> 16).astype(np.uint16).view(np.uint8)
    got = c.run(va, 2)
    for b in range(2):
        for i in range(Q):
            if not int(c.mask[b, i]) >> j & 1:
                assert (got[b, i].view(np.uint16) == clean[b, i].view(np.uint16)).all()
            elif what == "nan":
                assert np.isnan(got[b, i]).all()
