"""The five cache operators back to back in one replayed graph, nothing of torch's between them: each
call reads lengths, tables and rows that the call ahead of it has written, lengths in turn in two
buffers. Against the same steps on the host, byte for byte where rows and integers are concerned. No
reference counterpart."""
import numpy as np
import pytest

from tests import cache_ref as R
from tests.test_gpu_cache_ops import Pool, expect_rows, i32
from tests.test_gpu_tree import bound

pytestmark = pytest.mark.gpu
B, HQ, HKV, Q, D, PAGE, MP, PAGES = 5, 8, 2, 4, 128, 16, 24, 140


class Host:
    """The same state, stepped with plain restatements."""

    def __init__(self, pool, oracle):
        self.pool, self.oracle = pool, oracle

    def append(self, table, pos, k, v, nodes):
        at = 0
        for b in range(B):
            for i in range(int(nodes[b])):
                p = int(pos[b]) + i
                for side, x in ((0, k), (1, v)):
                    c, s = expect_rows(self.oracle, x[at], self.pool.fmt)
                    self.pool.host[side][0, table[b, p // PAGE], :, p % PAGE] = c
                    if s is not None:
                        self.pool.host[2 + side][0, table[b, p // PAGE], :, p % PAGE] = s
                at += 1

    def accept(self, table, lens, nodes, path, accepted):
        for h in self.pool.host:
            old = h.copy()
            for b in range(B):
                c = int(lens[b] - nodes[b])
                for i in range(int(accepted[b])):
                    s, d = c + int(path[b, i]), c + i
                    h[0, table[b, d // PAGE], :, d % PAGE] = old[0, table[b, s // PAGE], :, s % PAGE]
        return lens - nodes + accepted

    def tree(self, q, table, lens, nodes, mask):
        fmt, h = self.pool.fmt, self.pool.host
        out, mag = np.zeros((B, Q, HQ, D)), np.zeros((B, Q, HQ, D))
        G = HQ // HKV
        for b in range(B):
            L, n = int(lens[b]), min(int(nodes[b]), int(lens[b]))
            ids = table[b, :-(-L // PAGE)]
            for j in range(HKV):
                side = []
                for s in (0, 1):
                    c = np.ascontiguousarray(h[s][0, ids, j].reshape(-1, h[s].shape[-1])[:L])
                    sc = np.ascontiguousarray(h[2 + s][0, ids, j].reshape(-1, D // 64 * 2)[:L]).view(np.float16) if len(h) > 2 else None
                    side.append(R.values(c, sc, fmt))
                out[b, :n, j * G:j * G + G], mag[b, :n, j * G:j * G + G] = R.tree_attention(
                    q[b, :n, j * G:j * G + G].astype(np.float64), side[0], side[1], L - n, n, mask[b])
        return out, mag


@pytest.mark.parametrize("fmt", ["q4+", "q8+", "f16+", "bf16+"])
def test_five_calls_in_a_row(oracle, fmt):
    import torch
    import voltattn_b200 as va
    rng = np.random.default_rng(len(fmt))
    pool = Pool(fmt, PAGES, HKV, PAGE, D)
    for h in pool.host:  # (finite scales and entries of about 1 from the start)
        h[:] = 0
    lens = rng.integers(0, 60, B)
    table = R.make_table(rng, -(-lens // PAGE), MP, PAGES)
    refs = np.zeros(PAGES, np.int32)
    refs[table[table >= 0]] = 1
    x, s = R.random_rows(rng, PAGES * HKV * PAGE, D, fmt)
    for side in (0, 1):
        pool.host[side][:] = x.reshape(pool.host[side].shape)
        if s is not None:
            pool.host[2 + side][:] = np.ascontiguousarray(s).view(np.uint8).reshape(pool.host[2 + side].shape)
    pool.gpu = [torch.from_numpy(h.copy()).cuda() for h in pool.host]
    host = Host(pool, oracle)
    z = lambda *n: torch.zeros(*n, dtype=torch.int32, device="cuda")  # noqa: E731
    # one allocation for all small arrays: outputs lie next to inputs
    ints = torch.zeros(4096 + 6 * PAGES + 8 * B * MP, dtype=torch.int32, device="cuda")
    at = [0]

    def carve(*shape):
        n = int(np.prod(shape))
        at[0] += n
        return ints[at[0] - n:at[0]].view(shape)

    state = [(carve(PAGES), carve(B, MP), carve(B)) for _ in range(3)]
    accepted_lens = [carve(B), carve(B)]
    full, nodes, accepted = [carve(B), carve(B)], [carve(B), carve(B)], [carve(B), carve(B)]
    path, parent, short, used = [carve(B, Q), carve(B, Q)], [carve(B), carve(B)], carve(2), carve(1)
    cu = [carve(B + 1), carve(B + 1)]
    T = B * Q
    kv = [torch.zeros(T, 2 * HKV, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    q = torch.from_numpy(rng.standard_normal((B, Q, HQ, D)).astype(np.float16)).cuda()
    masks = [torch.zeros(B, Q, dtype=torch.int64, device="cuda") for _ in range(2)]
    chain = np.array([[(2 << i) - 1 for i in range(Q)]] * B, np.uint64)
    chain_t = torch.from_numpy(chain.view(np.int64)).cuda()
    outs = [torch.zeros(B, Q, HQ, D, dtype=torch.float16, device="cuda") for _ in range(5)]
    ws = torch.zeros(va.tree_workspace_bytes(B, HQ, HKV, Q, D, 4), dtype=torch.uint8, device="cuda")
    scratch = torch.zeros(va.pages_workspace_bytes(B, MP, PAGES), dtype=torch.uint8, device="cuda")
    g4 = (pool.gpu + [None, None])[:4]

    def bufs(out=None, w=None):
        return va.DeviceBufs(g4[0], g4[1], g4[2], g4[3], q, out, ws if w is None else w)

    def tree(mask, lens, nodes, table, out):
        va.decode_tree(fmt, bufs(out), mask, lens, nodes, table, MP, B, HQ, HKV, Q, PAGE, PAGES, D, S=3)

    def step():
        (r0, t0, l0), (r1, t1, l1), (r2, t2, _) = state
        va.fork_pages(fmt, bufs(w=scratch), r0, t0, l0, parent[0], r1, t1, l1, short[:1], B, B, MP, 2 * Q, HKV, PAGE, PAGES, D)
        where = l1
        for i in range(2):
            va.append_packed(fmt, kv[i][:, :HKV], kv[i][:, HKV:], bufs(), t1, MP, cu[i], where, B, HKV, PAGE, PAGES, D)
            tree(masks[i], full[i], nodes[i], t1, outs[2 * i])
            va.accept_tree(fmt, bufs(), t1, MP, full[i], nodes[i], path[i], accepted[i], accepted_lens[i], B, Q, HKV, PAGE, PAGES, D)
            where = accepted_lens[i]
            tree(chain_t, where, None, t1, outs[2 * i + 1])  # the lengths that were just written
        va.compact_pages(fmt, bufs(w=scratch), r1, t1, r2, t2, used, B, MP, HKV, PAGE, PAGES, D)
        tree(chain_t, where, None, t2, outs[4])
        va.fork_pages(fmt, bufs(w=scratch), r2, t2, where, parent[1], r0, t0, l0, short[1:], B, B, MP, 0, HKV, PAGE, PAGES, D)

    state[0][0].copy_(i32(refs)); state[0][1].copy_(i32(table)); state[0][2].copy_(i32(lens))  # noqa: E702
    start = [t.clone() for t in pool.gpu] + [ints.clone()]
    torch.cuda.synchronize()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        step()
        with torch.cuda.graph(graph, stream=stream):
            step()
    torch.cuda.synchronize()
    for t, v in zip(pool.gpu + [ints], start):
        t.copy_(v)
    qn = q.cpu().numpy()
    for turn in range(3):
        # this turn's trees, rows, paths and parents, and what the host makes of them
        par = [rng.integers(-1, B, B), rng.integers(0, B, B)]
        par[1][0] = 0
        n = [np.where(par[0] >= 0, rng.integers(0, Q + 1, B), 0) for _ in range(2)]  # (an empty slot has no pages)
        expect = []
        r1, t1, l1, sh, copies = R.fork(refs, table, lens, par[0], MP, PAGE, 2 * Q)
        assert sh == 0
        for f, t, rows in copies:
            for h in pool.host:
                h[:, t, :, :rows] = h[:, f, :, :rows]
        where = l1.astype(np.int64)
        for i in range(2):
            rows = torch.from_numpy(rng.standard_normal((T, 2 * HKV, D)).astype(np.float32)).to(torch.bfloat16)
            kv[i].copy_(rows)
            mask = R.random_tree(rng, B, Q)
            masks[i].copy_(torch.from_numpy(mask.view(np.int64)))
            rf = rows.float().numpy()
            host.append(t1, where, rf[:, :HKV], rf[:, HKV:], n[i])
            fl = where + n[i]
            expect.append(host.tree(qn, t1, fl, n[i], mask))
            acc, pa = np.zeros(B, int), np.full((B, Q), -1)
            for b in range(B):
                acc[b] = rng.integers(0, n[i][b] + 1)
                pa[b, :acc[b]] = np.sort(rng.choice(int(n[i][b]), acc[b], replace=False)) if acc[b] else []
            cu[i].copy_(i32(np.concatenate([[0], np.cumsum(n[i])])))
            full[i].copy_(i32(fl)); nodes[i].copy_(i32(n[i])); path[i].copy_(i32(pa)); accepted[i].copy_(i32(acc))  # noqa: E702
            where = host.accept(t1, fl, n[i], pa, acc)
            expect.append(host.tree(qn, t1, where, np.full(B, Q), chain))
        r2, t2, count, moves = R.compact(r1, t1)
        for h in pool.host:
            for f, t in moves:
                h[:, t] = h[:, f]
        expect.append(host.tree(qn, t2, where, np.full(B, Q), chain))
        refs, table, lens, sh, copies = R.fork(r2, t2, where, par[1], MP, PAGE, 0)
        assert sh == 0
        for f, t, rows in copies:
            for h in pool.host:
                h[:, t, :, :rows] = h[:, f, :, :rows]
        for i in range(2):
            parent[i].copy_(i32(par[i]))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        assert (state[0][0].cpu().numpy() == refs).all() and (state[0][1].cpu().numpy() == table).all()
        assert (state[0][2].cpu().numpy() == lens).all() and int(used) == count and not short.any()
        pool.check()
        for got, (want, mag) in zip(outs, expect):
            assert (np.abs(got.cpu().numpy().astype(np.float64) - want) <= bound(want, mag)).all()
