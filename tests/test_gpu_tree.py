"""Tree attention over a paged cache (va_decode_tree) against the definition in
64 bits, at the shapes and masks where it can go wrong. No reference
counterpart: the reference decodes one token at a time.

The bound, from the arithmetic: the weights are rounded once to fp16 (relative
2^-11 each, so at most 2^-11 * sum w |V| on an output), the output once more
(2^-11 of itself, or half of fp16's smallest step), and fp32 scores of size below
40 with errors of a few 2^-24 and the 2-ulp exponential change a weight by less
than 1e-5 of itself, numerator and denominator. bf16 / f16 rows are exact."""
import numpy as np
import pytest

from tests import cache_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def va():
    import torch
    assert torch.cuda.is_available()
    import voltattn_b200
    return voltattn_b200


def bound(out, mag):
    return 2.0 ** -11 * (np.abs(out) + mag) * 1.001 + 2e-5 * mag + 2.0 ** -25


class Case:
    """A pool with the sequences' pages at random places among pages of junk (nan
    scales, or rows of random bits), their trees, and the values expected."""

    def __init__(self, fmt, B, Hq, Hkv, Q, D, page, lens, nodes=None, seed=0, spare=3, mask=None, spread=1.0):
        import torch
        rng = np.random.default_rng([seed, B, Hq, Q, D, page])
        self.fmt, self.B, self.Hq, self.Hkv, self.Q, self.D, self.page = fmt, B, Hq, Hkv, Q, D, page
        self.lens = np.asarray(lens, np.int32)
        self.nodes = np.asarray(nodes if nodes is not None else [min(Q, l) for l in lens], np.int32)
        need = -(-self.lens // page)
        self.max_pages = max(1, int(need.max()))
        self.pages = int(need.sum()) + spare
        self.table = R.make_table(rng, need, self.max_pages, self.pages)
        self.mask = R.random_tree(rng, B, Q) if mask is None else mask
        rb, self.sides = R.row_bytes(fmt, D), []
        used = np.zeros((self.pages, page), bool)
        for b in range(B):
            for j in range(int(self.lens[b])):
                used[self.table[b, j // page], j % page] = True
        dead = np.repeat(~used[:, None], Hkv, 1)  # [pages, Hkv, page]
        for junk in (np.nan, np.inf):
            c, s = R.random_rows(rng, self.pages * Hkv * page, D, fmt, spread)
            c = c.reshape(self.pages, Hkv, page, rb).copy()
            c[dead] = rng.integers(0, 256, (int(dead.sum()), rb))
            if s is not None:
                s = s.reshape(self.pages, Hkv, page, D // 64).copy()
                s[dead] = junk
            self.sides.append([c, s])
        self.q = rng.standard_normal((B, Q, Hq, D)).astype(np.float16)
        self.dev = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()

    def rows(self, side, b, h):
        """float64 rows of sequence b, head h."""
        c, s = self.sides[side]
        L = int(self.lens[b])
        ids = self.table[b, :-(-L // self.page)]
        cc = np.ascontiguousarray(c[ids, h].reshape(-1, c.shape[-1])[:L])
        ss = None if s is None else s[ids, h].reshape(-1, s.shape[-1])[:L]
        return R.values(cc, ss, self.fmt)

    def expect(self):
        out = np.zeros((self.B, self.Q, self.Hq, self.D))
        mag = np.zeros_like(out)
        G = self.Hq // self.Hkv
        for b in range(self.B):
            n = int(self.nodes[b])
            for h in range(self.Hkv):
                hs = slice(h * G, h * G + G)
                o, m = R.tree_attention(self.q[b, :n, hs].astype(np.float64), self.rows(0, b, h), self.rows(1, b, h),
                                        int(self.lens[b]) - n, n, self.mask[b])
                out[b, :n, hs], mag[b, :n, hs] = o, m
        return out, mag

    def bufs(self, va, S=4, ws=None):
        import torch
        d = [self.dev(x) for side in self.sides for x in side]
        d = [x.view(torch.uint8) if i % 2 == 0 else x for i, x in enumerate(d)]
        q = self.dev(self.q)
        out = torch.full(self.q.shape, float("nan"), dtype=torch.float16, device="cuda")
        if ws is None:
            ws = torch.zeros(va.tree_workspace_bytes(self.B, self.Hq, self.Hkv, self.Q, self.D, max(S, 1)),
                             dtype=torch.uint8, device="cuda")
        return va.DeviceBufs(d[0], d[2], d[1], d[3], q, out, ws)

    def args(self):
        import torch
        return (self.dev(self.mask.view(np.int64)), self.dev(self.lens), self.dev(self.nodes), self.dev(self.table),
                self.max_pages, self.B, self.Hq, self.Hkv, self.Q, self.page, self.pages, self.D)

    def run(self, va, S=4, ws=None):
        import torch
        b = self.bufs(va, S, ws)
        va.decode_tree(self.fmt, b, *self.args(), S=S)
        torch.cuda.synchronize()
        return b.out.cpu().numpy()

    def check(self, va, S=4, ws=None):
        got = self.run(va, S, ws).astype(np.float64)
        want, mag = self.expect()
        err = np.abs(got - want)
        bad = ~(err <= bound(want, mag))
        assert not bad.any(), f"{int(bad.sum())} of {bad.size} off, worst {np.nanmax(err / bound(want, mag)):.2f} of the bound"
        return got


SHAPES = [  # B, Hq, Hkv, Q, D, page, lens, S
    (1, 4, 1, 1, 128, 64, [1], 1),
    (2, 8, 2, 4, 128, 32, [300, 77], 3),
    (3, 6, 2, 5, 64, 8, [129, 5, 640], 4),      # three query heads per KV head, 8-row pages
    (1, 8, 8, 16, 128, 24, [1000], 8),          # pages that end inside a block
    (2, 12, 2, 6, 128, 16, [97, 513], 2),       # 36 query rows: a tile and a bit
    (1, 2, 2, 33, 64, 256, [200], 1),
    (2, 16, 2, 8, 128, 64, [1500, 40], 16),     # 64 query rows
    (1, 16, 2, 64, 128, 40, [700], 3),          # 512 query rows, every bit of the mask
    (4, 3, 1, 7, 64, 128, [31, 32, 33, 128], 5),
]


@pytest.mark.parametrize("fmt", R.FORMATS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "B{}_Hq{}_Hkv{}_Q{}_D{}_P{}".format(*s[:6]))
def test_tree(va, fmt, shape):
    B, Hq, Hkv, Q, D, page, lens, S = shape
    Case(fmt, B, Hq, Hkv, Q, D, page, lens).check(va, S)


@pytest.mark.parametrize("fmt", ["q4+", "f16+"])
@pytest.mark.parametrize("Q", [1, 3, 12])
def test_lengths(va, fmt, Q):
    """No rows, one row, no context, unused slots, ragged trees, around every block edge."""
    lens = [0, 1, Q, Q + 1, 15, 16, 17, 31, 32, 33, 127, 128, 129, 255, 257, 511]
    nodes = [min(l, max(0, Q - i % 3)) for i, l in enumerate(lens)]
    for S in (1, 3, 0):
        Case(fmt, len(lens), 8, 4, Q, 128, 64, lens, nodes, seed=S).check(va, S)


@pytest.mark.parametrize("fmt", R.FORMATS)
@pytest.mark.parametrize("rows", [8, 40, 160])
def test_rows_that_see_nothing(va, fmt, rows):
    """Masks that leave a row empty, with and without rows before the drafted ones."""
    Q = max(4, rows // 4)
    mask = np.zeros((3, Q), np.uint64)
    mask[:, 1] = np.uint64(1 << (Q - 1))
    mask[2] = np.uint64(2 ** Q - 1)
    c = Case(fmt, 3, 4, 1, Q, 128, 32, [Q, Q + 50, Q], mask=mask)
    got = c.check(va, 2)
    assert (got[0, 0] == 0).all() and (got[0, 2:] == 0).all()


@pytest.mark.parametrize("fmt", R.FORMATS)
@pytest.mark.parametrize("G", [1, 4, 16])
@pytest.mark.parametrize("what", ["nan", "inf", "-inf"])
def test_unseen_rows_have_no_influence(va, fmt, G, what):
    """A drafted row of inf / nan (its entries, or its scales) reaches only the rows that see it."""
    Q, D = 10, 128
    c = Case(fmt, 2, 2 * G, 2, Q, D, 32, [150, Q])
    clean = c.run(va, 2)
    bad = float(what)
    j = 4  # node 4: seen by itself and its descendants
    for b in range(2):
        r = int(c.lens[b]) - Q + j
        for codes, scales in c.sides:
            at = (c.table[b, r // 32], slice(None), r % 32)
            if scales is not None:
                scales[at] = bad
            elif fmt == "f16+":
                codes[at] = np.broadcast_to(np.full(D, bad, np.float16).view(np.uint8), codes[at].shape)
            else:
                codes[at] = np.broadcast_to((np.full(D, bad, np.float32).view(np.uint32) >> 16).astype(np.uint16).view(np.uint8), codes[at].shape)
    got = c.run(va, 2)
    for b in range(2):
        for i in range(Q):
            sees = bool(int(c.mask[b, i]) >> j & 1)
            if sees:
                # an infinite score can be the lowest: a weight of 0 next to others, and a row that
                # has no weight at all (only without rows before the drafted ones) gives 0
                none = (got[b, i] == 0).all(-1) & (what != "nan" and c.lens[b] == Q)
                assert (~np.isfinite(got[b, i]) | none[:, None]).all()
            else:
                want, mag = clean[b, i].astype(np.float64), 3.0  # |V| < 3 on average
                assert np.isfinite(got[b, i]).all()
                assert (np.abs(got[b, i] - want) <= 2.0 ** -9 * mag).all()


@pytest.mark.parametrize("fmt", ["f16+", "bf16+", "f8+"])
def test_entry_of_inf_reaches_its_dim_only(va, fmt):
    """One entry of a drafted V row is nan: only that dim, only of the nodes that see it."""
    Q, D, j, d = 6, 128, 2, 77
    c = Case(fmt, 1, 8, 2, Q, D, 32, [60])
    want, mag = c.expect()
    r = 60 - Q + j
    at = (c.table[0, r // 32], 0, r % 32)
    row = c.sides[1][0][at]
    if fmt == "f8+":
        row[d] = 0x7F
    else:
        row[2 * d:2 * d + 2] = np.array([0x7FFF if fmt == "f16+" else 0x7FC0], np.uint16).view(np.uint8)
    got = c.run(va, 2).astype(np.float64)
    for i in range(Q):
        sees = bool(int(c.mask[0, i]) >> j & 1)
        hit = np.zeros((8, D), bool)
        hit[:4, d] = sees
        assert np.isnan(got[0, i][hit]).all()
        keep = ~hit
        keep[:4, :] &= True
        assert (np.abs(got[0, i] - want[0, i]) <= bound(want[0, i], mag[0, i]))[keep].all()


@pytest.mark.parametrize("fmt,spread", [("q8+", 3e-4), ("q8+", 2000.0), ("q4+", 1e-3), ("q4+", 8000.0), ("q3+", 5000.0), ("f8+", 4000.0),
                                        ("f16+", 2e-3), ("bf16+", 1e-2)])
def test_scales_of_any_size(va, fmt, spread):
    """Small and large V: the weights keep their 11 bits whatever the scales are."""
    c = Case(fmt, 1, 8, 2, 4, 128, 32, [400], spread=spread)
    c.q[:] = (c.q.astype(np.float32) / max(1.0, spread)).astype(np.float16)
    c.check(va, 2)


@pytest.mark.parametrize("fmt", ["q4+", "f16+", "q3+"])
@pytest.mark.parametrize("Q", [4, 24])
def test_splits_and_repeats(va, fmt, Q):
    """Any split count gives the same values up to rounding, and every call the same bits; one
    workspace serves every shape."""
    import torch
    c = Case(fmt, 2, 8, 2, Q, 128, 64, [2100, 900])
    ws = torch.zeros(va.tree_workspace_bytes(2, 8, 2, 64, 128, 32), dtype=torch.uint8, device="cuda")
    small = Case(fmt, 7, 8, 8, 2, 64, 8, [300, 2, 9, 100, 5, 40, 1])
    for S in (1, 2, 5, 17, 0):
        first = c.check(va, S, ws)
        small.check(va, 3, ws)
        assert (c.run(va, S, ws).astype(np.float64) == first).all()


def test_nodes_default(va):
    import torch
    c = Case("q8+", 2, 4, 2, 3, 128, 32, [50, 90])
    b = c.bufs(va)
    a = list(c.args())
    a[2] = None
    va.decode_tree(c.fmt, b, *a, S=2)
    torch.cuda.synchronize()
    want, mag = c.expect()
    assert (np.abs(b.out.cpu().numpy() - want) <= bound(want, mag)).all()


def test_strides_streams_and_graphs(va):
    """q as a slice of a fused projection, out with another order of dimensions, on a stream of the
    caller's, captured in a graph."""
    import torch
    c = Case("q4+", 2, 8, 2, 5, 128, 32, [200, 333])
    want, mag = c.expect()
    b = c.bufs(va)
    fused = torch.full((2, 5, 12, 128), float("nan"), dtype=torch.float16, device="cuda")
    fused[:, :, 2:10] = b.q
    b.q = fused[:, :, 2:10]
    store = torch.full((2, 8, 5, 136), float("nan"), dtype=torch.float16, device="cuda")
    b.out = store[..., :128].transpose(1, 2)
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
    assert torch.isnan(store[..., 128:]).all()


def test_offsets_past_32_bits(va):
    """Pages behind the first 4 GiB of each buffer."""
    import torch
    c = Case("f16+", 1, 4, 2, 3, 128, 64, [100], spare=0)
    pages = (9 << 29) // (2 * 64 * 256)
    lo = pages - c.pages
    b = c.bufs(va)
    for name in ("K", "V"):
        big = torch.zeros(pages * 2 * 64 * 256, dtype=torch.uint8, device="cuda")
        src = getattr(b, name).reshape(-1)
        big[lo * 2 * 64 * 256:] = src
        setattr(b, name, big)
    a = list(c.args())
    a[3] = a[3] + lo
    a[10] = pages
    va.decode_tree(c.fmt, b, *a, S=2)
    torch.cuda.synchronize()
    want, mag = c.expect()
    assert (np.abs(b.out.cpu().numpy() - want) <= bound(want, mag)).all()


def test_chain_matches_multiquery(va):
    """A chain over a cache that the causal multi-query decode also reads."""
    import torch
    B, Hq, Hkv, Q, D, Lmax = 2, 8, 4, 4, 128, 512
    chain = np.array([[(2 << i) - 1 for i in range(Q)]] * B, np.uint64)
    c = Case("q4+", B, Hq, Hkv, Q, D, Lmax, [500, 123], spare=0, mask=chain)
    c.table[:] = np.arange(B).reshape(B, 1)
    got = c.check(va, 2)
    b = c.bufs(va)
    q = b.q.transpose(1, 2).contiguous()
    out = torch.empty_like(q)
    ws = torch.zeros(va.gqa_workspace_bytes(B, Hq * Q, D, 2), dtype=torch.uint8, device="cuda")
    sides = [x.clone() for x in (b.K, b.V)]
    sc = [torch.nan_to_num(x, nan=0.0, posinf=0.0) for x in (b.scK, b.scV)]
    va.decode_multiquery("q4+", va.DeviceBufs(*sides, *sc, q, out, ws), torch.from_numpy(c.lens).cuda(), B, Hq, Hkv, Q, Lmax, D, 2)
    torch.cuda.synchronize()
    assert np.abs(out.transpose(1, 2).cpu().numpy().astype(np.float64) - got).max() < 2e-2


@pytest.mark.parametrize("fmt", R.FORMATS)
@pytest.mark.parametrize("rows,D", [(64, 128), (65, 128), (66, 64), (96, 128), (128, 64), (128, 128), (129, 128), (130, 64), (256, 128),
                                    (257, 128), (320, 64)])
def test_row_tile_edges(va, fmt, rows, D):
    """Query rows around each tile size of the kernels, with a full, a ragged and an unused sequence."""
    Q = 64 if rows > 129 else 32 if rows % 32 == 0 else 13 if rows % 13 == 0 else 11 if rows % 11 == 0 else 3
    G = -(-rows // Q)
    c = Case(fmt, 3, G, 1, Q, D, 32, [Q + 300, Q // 2 + 65, 0], [Q, Q // 2, 0], seed=rows)
    got = c.check(va, 3)
    assert (got[2] == 0).all() and (got[1, Q // 2:] == 0).all()


@pytest.mark.parametrize("fmt", R.FORMATS)
@pytest.mark.parametrize("what", ["nan", "inf", "-inf"])
def test_unseen_rows_in_tiles_of_128(va, fmt, what):
    test_unseen_rows_have_no_influence(va, fmt, 8, what)


@pytest.mark.parametrize("fmt", ["f16+", "bf16+", "f8+"])
@pytest.mark.parametrize("Hq", [32, 96])
def test_entry_of_nan_in_large_tiles(va, fmt, Hq):
    """One nan entry of a drafted V row, tiles of 128 and 256 query rows."""
    Q, D, j, d = 6, 128, 2, 77
    c = Case(fmt, 1, Hq, 1 if Hq == 32 else 2, Q, D, 32, [200], seed=Hq)
    want, mag = c.expect()
    r = 200 - Q + j
    row = c.sides[1][0][(c.table[0, r // 32], 0, r % 32)]
    if fmt == "f8+":
        row[d] = 0x7F
    else:
        row[2 * d:2 * d + 2] = np.array([0x7FFF if fmt == "f16+" else 0x7FC0], np.uint16).view(np.uint8)
    got = c.run(va, 2).astype(np.float64)
    G = Hq // c.Hkv
    for i in range(Q):
        hit = np.zeros((Hq, D), bool)
        hit[:G, d] = bool(int(c.mask[0, i]) >> j & 1)
        assert np.isnan(got[0, i][hit]).all()
        assert (np.abs(got[0, i] - want[0, i]) <= bound(want[0, i], mag[0, i]))[~hit].all()


@pytest.mark.parametrize("fmt", ["q8+", "f16+", "q3+", "bf16+"])
@pytest.mark.parametrize("G,Q", [(4, 4), (4, 32), (8, 32)])
def test_growing_scores(va, fmt, G, Q):
    """Scores that rise along the cache: the running reference moves block after block, in every range."""
    c = Case(fmt, 1, G, 1, Q, 128, 64, [1500], seed=Q)
    kc, ks = c.sides[0]
    for p in range(1500 - Q):  # keys grow from 1 / 40 to 10 times as large
        at = (c.table[0, p // 64], 0, p % 64)
        f = 0.025 * 400.0 ** (p / 1500)
        if ks is not None:
            ks[at] = (ks[at].astype(np.float32) * f).astype(np.float16)
        elif fmt == "f16+":
            kc[at] = (kc[at].view(np.float16).astype(np.float32) * f).astype(np.float16).view(np.uint8)
        else:
            x = (kc[at].view(np.uint16).astype(np.uint32) << 16).view(np.float32) * np.float32(f)
            kc[at] = (x.view(np.uint32) >> 16).astype(np.uint16).view(np.uint8)
    for S in (1, 4):
        c.check(va, S)


def test_many_sequences(va):
    """More (sequence, KV head) pairs than a grid dimension holds; one row each."""
    import torch
    B, Hkv = 8200, 8
    c = Case("q8+", 1, 8, 8, 1, 64, 8, [3], spare=0)
    b = c.bufs(va)
    b.q = b.q.expand(B, 1, 8, 64).contiguous()
    b.out = torch.full((B, 1, 8, 64), float("nan"), dtype=torch.float16, device="cuda")
    rep = lambda t, *s: t.expand(B, *s).contiguous()  # noqa: E731
    m, lens, nodes, table = c.args()[:4]
    va.decode_tree("q8+", b, rep(m, 1), rep(lens), rep(nodes), rep(table, 1), 1, B, 8, Hkv, 1, 8, c.pages, 64, S=1)
    torch.cuda.synchronize()
    want, mag = c.expect()
    assert (np.abs(b.out.cpu().numpy().astype(np.float64) - want) <= bound(want, mag)).all()
