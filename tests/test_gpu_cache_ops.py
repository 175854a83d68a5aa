"""Rows and pages of a paged cache: packed appends (bit-exact with the quantizer),
accepted rows, forks and compactions, against plain restatements entry by
entry. No reference counterpart: the reference's cache is one contiguous buffer."""
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


class Pool:
    """A pool of random bytes, its copy on the host, and views of its rows."""

    def __init__(self, fmt, pages, Hkv, page, D, layers=1, seed=0):
        import torch
        rng = np.random.default_rng([seed, pages, Hkv, page, D])
        self.fmt, self.pages, self.Hkv, self.page, self.D, self.layers = fmt, pages, Hkv, page, D, layers
        sizes = [R.row_bytes(fmt, D)] * 2 + ([2 * (D // 64)] * 2 if fmt in R.SCALED else [])
        shape = (layers, pages, Hkv, page)
        self.host = [rng.integers(0, 256, shape + (s,)).astype(np.uint8) for s in sizes]
        self.gpu = [torch.from_numpy(h.copy()).cuda() for h in self.host]

    def bufs(self, va, ws=None):
        g = self.gpu + [None, None]
        return va.DeviceBufs(g[0], g[1], g[2], g[3], ws=ws)

    def check(self):
        for h, g in zip(self.host, self.gpu):
            assert (g.cpu().numpy() == h).all()


def i32(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


IN = ["float32", "float16", "bfloat16"]


def expect_rows(oracle, x, fmt):
    """Codes and scales of fp32 rows [n, D] by the oracle's quantizer."""
    n, D = x.shape
    f = np.ascontiguousarray(x, np.float32).reshape(-1)
    if fmt == "f16+":
        return oracle.f2h(f).view(np.uint8).reshape(n, -1), None
    if fmt == "bf16+":
        return oracle.f2bf(f).view(np.uint8).reshape(n, -1), None
    c, s = oracle.quantize_f8(f, 1, n, D) if fmt == "f8+" else oracle.quantize(f, 1, n, D, R.BITS[fmt])
    return c.view(np.uint8).reshape(n, -1), np.ascontiguousarray(s).view(np.uint8).reshape(n, -1)


@pytest.mark.parametrize("fmt", R.FORMATS)
@pytest.mark.parametrize("kind", IN)
@pytest.mark.parametrize("Hkv,D,page,counts", [(1, 64, 8, [1]), (2, 128, 32, [3, 0, 17, 1]), (3, 64, 5, [40, 2]), (8, 128, 64, [130, 7])])
def test_append_packed(va, oracle, fmt, kind, Hkv, D, page, counts):
    """Every byte of the pool: the new rows as the quantizer gives them, the others as they were. k and v are slices
    of one projection; the values include exact ties, zeros, a group of zeros, large and tiny ones."""
    import torch
    rng = np.random.default_rng([Hkv, D, page])
    B, T = len(counts), sum(counts) + 3  # three tokens of nobody's
    pos = rng.integers(0, 30, B)
    need = -(-(pos + counts) // page)
    mp = int(need.max())
    pool = Pool(fmt, int(need.sum()) + 2, Hkv, page, D)
    table = R.make_table(rng, need, mp, pool.pages)
    x = rng.standard_normal((T, 2 * Hkv + 1, D)).astype(np.float32)
    x[0, 0] = np.round(x[0, 0] * 4) / 2
    x[0, 0, 0] = 3.5
    x[0, 1] *= 1e-6
    x[T // 2, :, :64] = 0
    x[-4] *= 3000
    xt = torch.from_numpy(x).to(getattr(torch, kind)).cuda()
    cu = np.concatenate([[0], np.cumsum(counts)])
    va.append_packed(fmt, xt[:, :Hkv], xt[:, Hkv:2 * Hkv], pool.bufs(va), i32(table), mp, i32(cu), i32(pos), B, Hkv, page, pool.pages, D)
    torch.cuda.synchronize()
    xf = xt.float().cpu().numpy()
    for side in range(2):
        for b in range(B):
            if not counts[b]:
                continue
            rows = xf[cu[b]:cu[b + 1], side * Hkv:(side + 1) * Hkv]
            c, s = expect_rows(oracle, rows.reshape(-1, D), fmt)
            for i in range(counts[b]):
                p = int(pos[b]) + i
                pool.host[side][0, table[b, p // page], :, p % page] = c.reshape(counts[b], Hkv, -1)[i]
                if s is not None:
                    pool.host[2 + side][0, table[b, p // page], :, p % page] = s.reshape(counts[b], Hkv, -1)[i]
    pool.check()


@pytest.mark.parametrize("fmt", ["q8+", "q4+", "q3+", "f8+"])
def test_append_odd_values(va, oracle, fmt):
    """nan, inf, values whose scale under- or overflows fp16, and quotients next to the rounding boundary."""
    import torch
    D, n = 128, 64
    rng = np.random.default_rng(5)
    x = rng.standard_normal((n, 1, D)).astype(np.float32)
    x[0, 0, 3], x[1, 0, 70], x[2, 0, 5] = np.nan, np.inf, -np.inf
    x[3] *= 1e-9
    x[4] *= 1e30
    x[5] *= 1e38
    x[6, 0, 0] = np.finfo(np.float32).max
    x[7] *= 1e-42
    for r in range(8, n):  # multiples of half a step, and one ulp around them
        step = np.float32(np.float16(rng.random() + 0.1))
        x[r, 0] = step * (rng.integers(-14, 15, D) / 2).astype(np.float32)
        x[r, 0, ::64] = step * {"q8+": 127, "q4+": 7, "q3+": 3, "f8+": 448}[fmt]
        x[r, 0, 1::2] = np.nextafter(x[r, 0, 1::2], np.float32(rng.choice([-9, 9])))
    pool = Pool(fmt, 4, 1, 16, D)
    xt = torch.from_numpy(x).cuda()
    va.append_packed(fmt, xt, xt, pool.bufs(va), i32([[2, 0, 3, 1]]), 4, i32([0, n]), i32([0]), 1, 1, 16, 4, D)
    torch.cuda.synchronize()
    c, s = expect_rows(oracle, x.reshape(n, D), fmt)
    order = [2, 0, 3, 1]
    for side in range(2):
        pool.host[side][0, order, 0] = c.reshape(4, 16, -1)
        pool.host[2 + side][0, order, 0] = s.reshape(4, 16, -1)
    pool.check()


def test_append_skips_what_has_no_page(va):
    """Rows past the table, entries outside the pool, negative positions, no tokens at all."""
    import torch
    pool = Pool("q4+", 3, 2, 16, 128)
    x = torch.randn(40, 2, 128, device="cuda")
    for table, pos, cu in (([[-1, 7]], [0], [0, 40]), ([[0, 1]], [-50], [0, 40]), ([[0, 1]], [32], [0, 40]),
                           ([[0, 1]], [0], [40, 40]), ([[0, 1]], [2 ** 31 - 1], [0, 40])):
        va.append_packed("q4+", x, x, pool.bufs(va), i32(table), 2, i32(cu), i32(pos), 1, 2, 16, 3, 128)
    va.append_packed("q4+", x[:0], x[:0], pool.bufs(va), i32([[0, 1]]), 2, i32([0, 0]), i32([0]), 1, 2, 16, 3, 128)
    torch.cuda.synchronize()
    pool.check()


@pytest.mark.parametrize("fmt", R.FORMATS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("P,page,layers", [(1, 8, 1), (9, 24, 2), (64, 64, 3), (33, 7, 1)])
def test_accept_tree(va, fmt, D, P, page, layers):
    import torch
    rng = np.random.default_rng([P, page])
    B, Hkv = 5, 3
    nodes = np.array([P, max(1, P // 2), P, 1, 0])
    lens = nodes + np.array([0, 13, 100, 40, 20])
    need = -(-lens // page)
    mp = int(need.max())
    pool = Pool(fmt, int(need.sum()) + 2, Hkv, page, D, layers)
    table = R.make_table(rng, need, mp, pool.pages)
    path = np.full((B, P), -1)
    accepted = np.zeros(B, int)
    for b in range(B):
        k = int(rng.integers(0, nodes[b] + 1))
        path[b, :k] = np.sort(rng.choice(int(nodes[b]), k, replace=False)) if k else []
        accepted[b] = k
    want = lens - nodes + accepted
    new = i32(np.zeros(B))
    va.accept_tree(fmt, pool.bufs(va), i32(table), mp, i32(lens), i32(nodes), i32(path), i32(accepted), new, B, P, Hkv, page,
                   pool.pages, D, layers=layers)
    torch.cuda.synchronize()
    assert (new.cpu().numpy() == want).all()
    for h in pool.host:
        old = h.copy()
        for b in range(B):
            c = int(lens[b] - nodes[b])
            for i in range(accepted[b]):
                s, d = c + int(path[b, i]), c + i
                h[:, table[b, d // page], :, d % page] = old[:, table[b, s // page], :, s % page]
    pool.check()


def test_accept_ends_at_a_bad_entry(va):
    """Paths that do not ascend, leave the tree, or are longer than it: cut there."""
    import torch
    paths = [[0, 2, 2, 3], [1, 0, 2, 3], [0, 9, 1, 2], [-1, 1, 2, 3], [0, 1, 2, 3], [1, 3, -1, 0]]
    accepted, want = [4, 4, 4, 4, 99, -3], [2, 1, 1, 0, 4, 0]
    B = len(paths)
    pool = Pool("q8+", B, 1, 16, 64)
    table = np.arange(B).reshape(B, 1)
    lens, nodes = np.full(B, 10), np.full(B, 5)
    new = i32(np.zeros(B))
    va.accept_tree("q8+", pool.bufs(va), i32(table), 1, i32(lens), i32(nodes), i32(paths), i32(accepted), new, B, 4, 1, 16, B, 64)
    torch.cuda.synchronize()
    assert (new.cpu().numpy() == 5 + np.array(want)).all()
    for h in pool.host:
        old = h.copy()
        for b in range(B):
            for i in range(want[b]):
                h[0, b, 0, 5 + i] = old[0, b, 0, 5 + paths[b][i]]
    pool.check()


def fork_case(rng, B, page, reserve, spare, shared):
    lens = rng.integers(0, 6 * page, B)
    lens[0] = 2 * page  # a full last page
    held = -(-lens // page) + (rng.random(B) < 0.3)  # some hold a page ahead
    mp = int(held.max()) + 1
    pages = int(held.sum()) + spare
    table = R.make_table(rng, held, mp, pages)
    refs = np.zeros(pages, np.int32)
    refs[table[table >= 0]] = 1
    if shared and B > 2 and lens[0] >= page and lens[1] >= page:  # a page that two sequences already share
        refs[table[1, 0]] -= 1
        table[1, 0] = table[0, 0]
        refs[table[0, 0]] += 1
    return lens, table, refs, mp, pages


@pytest.mark.parametrize("fmt", R.FORMATS)
@pytest.mark.parametrize("B,Bout,page,reserve,spare,layers,D", [
    (1, 1, 8, 0, 0, 1, 128), (1, 5, 16, 1, 20, 2, 64), (6, 6, 24, 30, 3, 1, 128), (6, 9, 32, 0, 40, 3, 64), (40, 70, 64, 5, 200, 2, 128),
    (5, 2, 8, 9, 0, 1, 64)])
def test_fork_pages(va, fmt, B, Bout, page, reserve, spare, layers, D):
    """Parents several times, once and never; too few free pages; a page that is shared already."""
    import torch
    rng = np.random.default_rng([B, Bout, page])
    lens, table, refs, mp, pages = fork_case(rng, B, page, reserve, spare, True)
    parent = rng.integers(-1, B, Bout)
    parent[-1] = 0
    pool = Pool(fmt, pages, 2, page, D, layers)
    ws = torch.zeros(va.pages_workspace_bytes(Bout, mp, pages), dtype=torch.uint8, device="cuda")
    nr, nt, nl, sh = i32(np.zeros(pages)), i32(np.zeros((Bout, mp))), i32(np.zeros(Bout)), i32([9])
    va.fork_pages(fmt, pool.bufs(va, ws), i32(refs), i32(table), i32(lens), i32(parent), nr, nt, nl, sh, B, Bout, mp, reserve, 2, page,
                  pages, D, layers=layers)
    torch.cuda.synchronize()
    wr, wt, wl, short, copies = R.fork(refs, table, lens, parent, mp, page, reserve)
    assert int(sh.cpu()[0]) == short
    assert (nt.cpu().numpy() == wt).all() and (nl.cpu().numpy() == wl).all() and (nr.cpu().numpy() == wr).all()
    assert (wr >= 0).all() and wr.sum() == (wt >= 0).sum()  # the counts are those of the new tables
    for h in pool.host:
        for f, t, rows in copies:
            h[:, t, :, :rows] = h[:, f, :, :rows]
    pool.check()


def test_fork_frees_everything(va):
    """No parent at all: every page is free again."""
    import torch
    rng = np.random.default_rng(3)
    lens, table, refs, mp, pages = fork_case(rng, 8, 16, 0, 5, True)
    pool = Pool("q4+", pages, 2, 16, 128)
    ws = torch.zeros(va.pages_workspace_bytes(8, mp, pages), dtype=torch.uint8, device="cuda")
    nr, nt, nl, sh = i32(np.ones(pages)), i32(np.zeros((8, mp))), i32(np.ones(8)), i32([9])
    va.fork_pages("q4+", pool.bufs(va, ws), i32(refs), i32(table), i32(lens), i32([-1] * 7 + [8]), nr, nt, nl, sh, 8, 8, mp, 100, 2, 16,
                  pages, 128)
    torch.cuda.synchronize()
    assert not nr.any() and not nl.any() and (nt == -1).all() and not sh.any()
    pool.check()


@pytest.mark.parametrize("fmt", R.FORMATS)
@pytest.mark.parametrize("pages,used,B,page,layers,D", [(1, 1, 1, 8, 1, 64), (7, 3, 2, 16, 2, 128), (100, 60, 9, 24, 1, 64),
                                                        (300, 299, 4, 8, 2, 128), (50, 0, 2, 8, 1, 64)])
def test_compact_pages(va, fmt, pages, used, B, page, layers, D):
    import torch
    rng = np.random.default_rng([pages, used])
    mp = max(1, -(-used // B))
    table = np.full((B, mp), -1, np.int32)
    table.reshape(-1)[:used] = rng.permutation(pages)[:used]
    refs = np.zeros(pages, np.int32)
    refs[table[table >= 0]] = rng.integers(1, 4, used)
    pool = Pool(fmt, pages, 2, page, D, layers)
    ws = torch.zeros(va.pages_workspace_bytes(B, mp, pages), dtype=torch.uint8, device="cuda")
    nr, nt, u = i32(np.zeros(pages)), i32(np.zeros((B, mp))), i32([77])
    va.compact_pages(fmt, pool.bufs(va, ws), i32(refs), i32(table), nr, nt, u, B, mp, 2, page, pages, D, layers=layers)
    torch.cuda.synchronize()
    wr, wt, n, moves = R.compact(refs, table)
    assert int(u.cpu()[0]) == n == used
    assert (nr.cpu().numpy() == wr).all() and (nt.cpu().numpy() == wt).all()
    for h in pool.host:
        for f, t in moves:
            h[:, t] = h[:, f]
    pool.check()


def test_many_pages(va):
    """Tens of thousands of pages (small ones), more than one pass of the plan's scan."""
    import torch
    rng = np.random.default_rng(1)
    pages, B, mp, page, D = 30011, 64, 400, 8, 64
    pool = Pool("q4+", pages, 1, page, D)
    lens = rng.integers(0, (mp - 2) * page, B)
    held = -(-lens // page)
    table = R.make_table(rng, held, mp, pages)
    refs = np.zeros(pages, np.int32)
    refs[table[table >= 0]] = 1
    parent = rng.integers(-1, B, B)
    ws = torch.zeros(va.pages_workspace_bytes(B, mp, pages), dtype=torch.uint8, device="cuda")
    nr, nt, nl, sh = i32(np.zeros(pages)), i32(np.zeros((B, mp))), i32(np.zeros(B)), i32([9])
    va.fork_pages("q4+", pool.bufs(va, ws), i32(refs), i32(table), i32(lens), i32(parent), nr, nt, nl, sh, B, B, mp, 100, 1, page, pages, D)
    cr, ct, u = i32(np.zeros(pages)), i32(np.zeros((B, mp))), i32([0])
    va.compact_pages("q4+", pool.bufs(va, ws), nr, nt, cr, ct, u, B, mp, 1, page, pages, D)
    torch.cuda.synchronize()
    wr, wt, wl, short, copies = R.fork(refs, table, lens, parent, mp, page, 100)
    assert (nt.cpu().numpy() == wt).all() and (nl.cpu().numpy() == wl).all() and (nr.cpu().numpy() == wr).all()
    r2, t2, n, moves = R.compact(wr, wt)
    assert (cr.cpu().numpy() == r2).all() and (ct.cpu().numpy() == t2).all() and int(u.cpu()[0]) == n
    for h in pool.host:
        for f, t, rows in copies:
            h[:, t, :, :rows] = h[:, f, :, :rows]
        for f, t in moves:
            h[:, t] = h[:, f]
    pool.check()
