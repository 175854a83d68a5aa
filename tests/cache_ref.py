"""Plain restatements, in 64 bits, of the operators over a paged cache: rows of
every format, tree attention, packed appends, accepted rows, forks and
compactions. Written from the definitions in include/voltattn.h; no code of the
package is used. Shared by the tests of these operators."""
import numpy as np

BITS = {"f16+": 16, "bf16+": 16, "f8+": 8, "q8+": 8, "q4+": 4, "q3+": 3}
SCALED = ("f8+", "q8+", "q4+", "q3+")
FORMATS = list(BITS)


def row_bytes(fmt, D):
    return D * BITS[fmt] // 8


def values(codes, scales, fmt):
    """float64 values of rows: codes uint8 [n, bytes], scales float16 [n, D/64] or None."""
    if fmt == "f16+":
        return codes.view(np.float16).astype(np.float64)
    if fmt == "bf16+":
        return (codes.view(np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    if fmt == "f8+":
        e, m = (codes >> 3 & 15).astype(np.int64), (codes & 7).astype(np.float64)
        v = np.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * 2.0 ** (e - 7.0)) * np.where(codes & 128, -1.0, 1.0)
        v = np.where((codes & 127) == 127, np.nan, v)
    elif fmt == "q8+":
        v = codes.view(np.int8).astype(np.float64)
    else:
        k = BITS[fmt]
        bits = np.unpackbits(codes, axis=1, bitorder="little").reshape(codes.shape[0], codes.shape[1] * 8 // k, k).astype(np.float64)
        v = bits @ (2.0 ** np.arange(k)) - 2.0 ** (k - 1)
    with np.errstate(invalid="ignore", over="ignore"):
        return v * np.repeat(scales.astype(np.float64), 64, axis=1)


def random_rows(rng, n, D, fmt, spread=1.0):
    """Codes and scales of n rows with values of about N(0, spread)."""
    x = rng.standard_normal((n, D)) * spread
    if fmt == "f16+":
        return x.astype(np.float16).view(np.uint8), None
    if fmt == "bf16+":
        u = x.astype(np.float32).view(np.uint32)
        return (u >> 16).astype(np.uint16).view(np.uint8).reshape(n, 2 * D), None
    s = (np.abs(rng.standard_normal((n, D // 64))) * 0.3 + 0.7) * spread
    if fmt == "f8+":
        c = rng.integers(0, 256, (n, D)).astype(np.uint8)
        c = np.where((c & 127) == 127, 0, c).astype(np.uint8)
        return c, (s / 100).astype(np.float16)
    if fmt == "q8+":
        return rng.integers(-127, 128, (n, D)).astype(np.int8).view(np.uint8), (s / 60).astype(np.float16)
    lim = 7 if fmt == "q4+" else 3
    v = rng.integers(0, 2 * lim + 1, (n, D)) + 1  # field = code + lim + 1
    k = BITS[fmt]
    bits = (v[..., None] >> np.arange(k) & 1).astype(np.uint8).reshape(n, -1)
    return np.packbits(bits, axis=1, bitorder="little"), (s / lim * 2).astype(np.float16)


def make_table(rng, need, max_pages, num_pages):
    """Each sequence's pages at shuffled places of the pool, -1 past its last."""
    t = np.full((len(need), max_pages), -1, np.int32)
    perm, k = rng.permutation(num_pages), 0
    for b, n in enumerate(need):
        t[b, :n] = perm[k:k + n]
        k += n
    return t


def random_tree(rng, B, Q):
    """tree_mask [B][Q] of random trees: every node sees its ancestors and itself."""
    mask = np.zeros((B, Q), np.uint64)
    for b in range(B):
        for i in range(Q):
            par = int(rng.integers(-1, i)) if i else -1
            mask[b, i] = (mask[b, par] if par >= 0 else np.uint64(0)) | np.uint64(1 << i)
    return mask


def tree_attention(q, K, V, ctx, n, mask):
    """One sequence and KV head: q [rows, D] with node ids per row in `n`'s order, K / V [L, D] float64.
    q: [n, G, D]; returns out and the sums of weight * |V| [n, G, D] (rounding bounds)."""
    G, D = q.shape[1:]
    out, mag = np.zeros((n, G, D)), np.zeros((n, G, D))
    for i in range(n):
        rows = list(range(ctx)) + [ctx + j for j in range(n) if int(mask[i]) >> j & 1]
        if not rows:
            continue
        s = q[i] @ K[rows].T / np.sqrt(float(D))
        w = np.exp(s - s.max(1, keepdims=True))
        w /= w.sum(1, keepdims=True)
        out[i], mag[i] = w @ V[rows], w @ np.abs(V[rows])
    return out, mag


def fork(refs, table, lens, parent, max_pages, page_rows, reserve):
    """New refs, table, lens, shortage, and the copies [(from, to, rows)], entry by entry."""
    refs = refs.copy()
    free = [p for p in range(len(refs)) if refs[p] == 0]
    P, Bin, Bout = len(refs), len(lens), len(parent)
    kids = [sum(1 for x in parent if x == s) for s in range(Bin)]
    new_table = np.full((Bout, max_pages), -1, np.int32)
    new_lens = np.zeros(Bout, np.int32)
    copies, short, started = [], 0, set()
    new_refs = refs.copy()
    for s in range(Bin):
        for j in range(max_pages):
            e = table[s, j]
            if 0 <= e < P:
                new_refs[e] += kids[s] - 1 if j < lens[s] // page_rows else (0 if kids[s] else -1)
    for i, s in enumerate(parent):
        if not 0 <= s < Bin:
            continue
        keep = s not in started
        started.add(s)
        full, rest = divmod(int(lens[s]), page_rows)
        new_lens[i] = lens[s]
        for j in range(max_pages):
            e = table[s, j] if (keep or j < full) and 0 <= table[s, j] < P else -1
            if e < 0 and j < min(max_pages, -(-(int(lens[s]) + reserve) // page_rows)):
                if free:
                    e = free.pop(0)
                    new_refs[e] += 1
                    if j == full and rest and not keep:
                        copies.append((int(table[s, j]), e, -(-rest // 8) * 8))
                else:
                    short += 1
                    if j == full and rest:
                        new_lens[i] = full * page_rows
            new_table[i, j] = e
    return new_refs, new_table, new_lens, short, copies


def compact(refs, table):
    """New refs, table, the number in use and the moves [(from, to)]."""
    n = int((refs > 0).sum())
    holes = [p for p in range(n) if refs[p] <= 0]
    movers = [p for p in range(n, len(refs)) if refs[p] > 0]
    to = dict(zip(movers, holes))
    new = np.zeros_like(refs)
    for p in range(len(refs)):
        if refs[p] > 0:
            new[to.get(p, p)] = refs[p]
    return new, np.vectorize(lambda e: to.get(int(e), int(e)), otypes=[np.int32])(table), n, list(zip(movers, holes))
