"""What is measured of the speculative-decoding and page operators: the work of
one pass, its inputs, the plain form in elementary torch operations, the calls
of the framework, and the values in 64 bits.

Five operators over a paged, quantized KV cache:
  tree     decode_tree     attention of a tree of drafted tokens over the cache
  append   append_packed   K/V rows of packed tokens quantized into their pages
  step     append_packed + decode_tree + accept_tree: one verification step, whose
           accepted rows are moved together at the end of the sequence
  fork     fork_pages      sequences forked, reordered and freed, last pages copied
  compact  compact_pages   the pages in use moved to the front of the pool
"""
import numpy as np
import torch

own = False

DEV = "cuda"
BITS = {"f16+": 16, "bf16+": 16, "f8+": 8, "q8+": 8, "q4+": 4, "q3+": 3}
LIM = {"f8+": 448.0, "q8+": 127.0, "q4+": 7.0, "q3+": 3.0}
DTYPE = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
WS_BYTES = 64 << 20


# ---- cases ----------------------------------------------------------------------------------


def listed():
    t = {"op": "tree", "D": 128, "ragged": False}
    return [
        # one user's sequence, a short context, eight drafted tokens: latency counts
        {**t, "name": "tree_one_q4", "fmt": "q4+", "B": 1, "Hq": 32, "Hkv": 8, "Q": 8, "lo": 1000, "hi": 1024, "page": 64},
        # a chat server's batch, trees of up to 16 tokens, ragged contexts, 8-bit cache
        {**t, "name": "tree_chat_q8", "fmt": "q8+", "B": 16, "Hq": 32, "Hkv": 8, "Q": 16, "lo": 1024, "hi": 8192, "page": 64,
         "ragged": True},
        # long documents, 4-bit cache, trees of 32
        {**t, "name": "tree_long_q4", "fmt": "q4+", "B": 8, "Hq": 32, "Hkv": 8, "Q": 32, "lo": 16384, "hi": 32768, "page": 128},
        # the largest trees, eight query heads per KV head, 16-bit cache: the products count
        {**t, "name": "tree_wide_f16", "fmt": "f16+", "B": 16, "Hq": 32, "Hkv": 4, "Q": 64, "lo": 2048, "hi": 8192, "page": 32},
        # drafted tokens of a batch of trees, as a model's bf16 projection gives them
        {"name": "append_draft_q4", "op": "append", "fmt": "q4+", "in": "bf16", "B": 32, "Hkv": 8, "D": 128, "lo": 7, "hi": 16,
         "page": 64},
        # packed prompts of odd lengths into an 8-bit cache
        {"name": "append_prompt_q8", "op": "append", "fmt": "q8+", "in": "fp16", "B": 12, "Hkv": 8, "D": 128, "lo": 301,
         "hi": 4099, "page": 64},
        # a small model's verification step: 64-wide heads, three query heads per KV head
        {"name": "step_small_q8", "op": "step", "fmt": "q8+", "in": "fp16", "B": 4, "Hq": 12, "Hkv": 4, "D": 64, "Q": 5, "lo": 200,
         "hi": 900, "page": 16, "ragged": True},
        # a server's verification step, one KV head per query head, 3-bit cache
        {"name": "step_mha_q3", "op": "step", "fmt": "q3+", "in": "bf16", "B": 8, "Hq": 32, "Hkv": 32, "D": 128, "Q": 12,
         "lo": 1024, "hi": 6000, "page": 64, "ragged": True},
        # four beams each of a few requests, reordered after a token
        {"name": "fork_beams_q4", "op": "fork", "fmt": "q4+", "layers": 2, "B": 16, "Hkv": 8, "D": 128, "lo": 100, "hi": 2000,
         "page": 64, "spare": 64, "reserve": 1},
        # many samples forked from prompts over a whole model's cache
        {"name": "fork_samples_f16", "op": "fork", "fmt": "f16+", "layers": 4, "B": 96, "Hkv": 8, "D": 128, "lo": 200, "hi": 1500,
         "page": 128, "spare": 400, "reserve": 16},
        # a small pool after some requests have ended
        {"name": "compact_small_q8", "op": "compact", "fmt": "q8+", "layers": 2, "B": 8, "Hkv": 8, "D": 128, "pages": 200,
         "used": 120, "moved": 30, "page": 32},
        # a server's pool that is to be shrunk
        {"name": "compact_large_q4", "op": "compact", "fmt": "q4+", "layers": 4, "B": 64, "Hkv": 8, "D": 128, "pages": 6001,
         "used": 3500, "moved": 1400, "page": 64},
    ]


def _cost(c):
    w = work(c)
    return w["bytes"] / 6e12 + w["flops"] / 5e14


def draw(rng):
    def log(a, b):
        return int(round(a * (b / a) ** rng.random()))

    fmt = rng.choice(sorted(BITS))
    op = rng.choice(["tree", "tree", "tree", "append", "step", "fork", "compact"])
    g = rng.choice([1, 2, 3, 4, 6, 8])
    hkv = rng.choice([1, 2, 4, 8, 16] if g > 1 else [4, 8, 16, 32])
    page = rng.choice([8, 16, 24, 32, 64, 64, 128, 256])
    c = {"op": op, "fmt": fmt, "Hkv": hkv, "D": rng.choice([64, 128, 128]), "page": page}
    if op in ("tree", "step"):
        hi = log(16, 32768)
        c.update(B=log(1, 64), Hq=g * hkv, Q=log(1, 64), lo=max(0, int(hi * rng.random())), hi=hi, ragged=rng.random() < 0.5)
        if op == "step":
            c["in"] = rng.choice(sorted(DTYPE))
        while _cost(c) > 0.8 * _cost(listed()[3]):
            c["B"], c["lo"], c["hi"] = (c["B"] + 1) // 2, c["lo"] // 2, c["hi"] // 2
    elif op == "append":
        hi = log(1, 6000)
        c.update({"in": rng.choice(sorted(DTYPE)), "B": log(1, 64), "lo": int(hi * rng.random()), "hi": hi})
        while c["B"] * c["hi"] * c["Hkv"] * c["D"] > 30_000_000:
            c["B"] = (c["B"] + 1) // 2
            c["hi"], c["lo"] = max(1, c["hi"] // 2), c["lo"] // 2
    elif op == "fork":
        hi = log(10, 2000)
        c.update(layers=log(1, 16), B=log(1, 96), lo=int(hi * rng.random()), hi=hi, spare=0, reserve=log(1, 64))
        c["spare"] = c["B"] * (2 + c["reserve"] // page) + log(1, 100)
        while _pool_bytes(c, c["B"] * (hi // page + 1) + c["spare"]) > 6e8 and c["layers"] > 1:
            c["layers"] = (c["layers"] + 1) // 2
    else:
        pages = log(20, 6000)
        used = max(2, int(pages * (0.3 + 0.6 * rng.random())))
        c.update(layers=log(1, 8), B=log(1, 64), pages=pages, used=used, moved=int(min(used, pages - used) * rng.random()))
        while _pool_bytes(c, pages) > 6e8 and c["layers"] > 1:
            c["layers"] = (c["layers"] + 1) // 2
        while _pool_bytes(c, c["pages"]) > 6e8:
            c["pages"], c["used"], c["moved"] = c["pages"] // 2, max(2, c["used"] // 2), c["moved"] // 2
        c["moved"] = min(c["moved"], c["used"], c["pages"] - c["used"])
    return c


# ---- sizes ----------------------------------------------------------------------------------


def _row(c):
    """Bytes of one row's codes and scales."""
    return c["D"] * BITS[c["fmt"]] // 8, (2 * (c["D"] // 64) if c["fmt"] in LIM else 0)


def _pool_bytes(c, pages):
    return 2 * c.get("layers", 1) * pages * c["Hkv"] * c["page"] * sum(_row(c))


def _lens(c, lo=None, hi=None):
    """The sequences' lengths: spread over [lo, hi], the largest first."""
    lo, hi = c["lo"] if lo is None else lo, c["hi"] if hi is None else hi
    u = (np.arange(c["B"]) * 0.6180339887498949) % 1.0
    return (hi - np.floor((hi - lo + 1) * u).clip(0, hi - lo)).astype(np.int64)


def _nodes(c):
    """Drafted tokens of each sequence: Q, or ragged with one sequence that has all Q."""
    if not c["ragged"]:
        return np.full(c["B"], c["Q"], np.int64)
    return 1 + (c["Q"] - 1) - ((np.arange(c["B"]) * 7) % c["Q"])


def _parents(c, rng):
    """fork: which sequence each new one continues (-1: none). About half go on, some of those several times."""
    return np.where(rng.random(c["B"]) < 0.1, -1, (rng.random(c["B"]) ** 2 * c["B"]).astype(np.int64))


def work(case):
    c = case
    rb, sb = _row(c)
    row = 2 * (rb + sb)  # K and V
    if c["op"] in ("tree", "step"):
        ctx, n = _lens(c), _nodes(c)
        by = int((ctx + n).sum()) * c["Hkv"] * row + 2 * int(n.sum()) * c["Hq"] * c["D"] * 2 + 8 * int(n.sum())
        fl = 4 * c["Hq"] * c["D"] * int((n * (ctx + 1)).sum())
        if c["op"] == "step":  # the new rows in and out of the cache once
            by += int(n.sum()) * c["Hkv"] * (2 * c["D"] * DTYPE[c["in"]].itemsize + row)
        return {"bytes": by, "flops": fl}
    if c["op"] == "append":
        rows = int(_lens(c).sum()) * c["Hkv"]
        return {"bytes": rows * (2 * c["D"] * DTYPE[c["in"]].itemsize + row) + 8 * c["B"], "flops": 0}
    if c["op"] == "fork":  # tables and counts; about a third of the sequences copies half a page
        pages = int((_lens(c) // c["page"] + 1).sum()) + c["spare"]
        per = c["layers"] * c["Hkv"] * row * c["page"] // 2
        return {"bytes": 8 * pages + 8 * pages + 2 * (c["B"] // 3) * per, "flops": 0}
    return {"bytes": 16 * c["pages"] + 2 * c["moved"] * c["layers"] * c["Hkv"] * row * c["page"], "flops": 0}


# ---- inputs ---------------------------------------------------------------------------------


def _quantize(x, fmt):
    """Codes (bytes) and scales of rows x [..., D], by the framework's group rule."""
    if fmt == "f16+":
        return x.half().contiguous().view(torch.uint8), None
    if fmt == "bf16+":
        return x.bfloat16().contiguous().view(torch.uint8), None
    x = x.float()
    g = x.reshape(*x.shape[:-1], x.shape[-1] // 64, 64)
    amax = g.abs().amax(-1)
    s = torch.where(amax > 0, amax / LIM[fmt], torch.ones_like(amax)).half()
    y = g / s.float().unsqueeze(-1)
    if fmt == "f8+":
        return y.clamp(-448, 448).to(torch.float8_e4m3fn).reshape(x.shape).view(torch.uint8), s
    v = y.round().clamp(-LIM[fmt], LIM[fmt]).to(torch.int32).reshape(x.shape)
    if fmt == "q8+":
        return v.to(torch.int8).view(torch.uint8), s
    if fmt == "q4+":
        v = (v + 8).reshape(*x.shape[:-1], -1, 2)
        return (v[..., 0] | v[..., 1] << 4).to(torch.uint8), s
    v = (v + 4).reshape(*x.shape[:-1], -1, 8)
    w = v[..., 0] | v[..., 1] << 3 | v[..., 2] << 6 | v[..., 3] << 9 | v[..., 4] << 12 | v[..., 5] << 15 | v[..., 6] << 18 | v[..., 7] << 21
    return torch.stack((w & 255, w >> 8 & 255, w >> 16), -1).to(torch.uint8).reshape(*x.shape[:-1], -1), s


def _fill(c, gen, pages, outliers):
    """One side of the pool: codes [layers*pages*Hkv*page, bytes] and scales, of rows drawn N(0, 1); of K's entries
    1% are eight times as large."""
    rows = c.get("layers", 1) * pages * c["Hkv"] * c["page"]
    rb, sb = _row(c)
    codes = torch.empty(rows, rb, dtype=torch.uint8, device=DEV)
    scales = torch.empty(rows, sb // 2, dtype=torch.float16, device=DEV) if sb else None
    for r in range(0, rows, 1 << 20):
        n = min(1 << 20, rows - r)
        x = torch.randn(n, c["D"], generator=gen, device=DEV)
        if outliers:
            x = torch.where(torch.rand(n, c["D"], generator=gen, device=DEV) < 0.01, 8 * x, x)
        k, s = _quantize(x, c["fmt"])
        codes[r:r + n] = k
        if sb:
            scales[r:r + n] = s
    return codes, scales


def _table(rng, need, max_pages, pages):
    """Each sequence's pages at random places of the pool; -1 past its last."""
    table = np.full((len(need), max_pages), -1, np.int32)
    perm, k = rng.permutation(pages), 0
    for b, n in enumerate(need):
        table[b, :n] = perm[k:k + n]
        k += n
    return table


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEV)


def prepare(case, seed):
    c = case
    rng = np.random.default_rng([seed, 11])
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    st = {"case": c, "ws": torch.zeros(WS_BYTES, dtype=torch.uint8, device=DEV)}
    if c["op"] == "compact":
        # `used` pages, `moved` of them past the front; shared by the sequences at random, a few more than once
        low = rng.permutation(c["used"])[:c["used"] - c["moved"]]
        high = c["used"] + rng.permutation(c["pages"] - c["used"])[:c["moved"]]
        pages = rng.permutation(np.concatenate([low, high]))
        per = -(-c["used"] // c["B"])
        table = np.full((c["B"], per + 2), -1, np.int32)
        refs = np.zeros(c["pages"], np.int32)
        for b in range(c["B"]):
            mine = pages[b * per:(b + 1) * per]
            table[b, :len(mine)] = mine
            refs[mine] += 1
        if c["B"] > 1 and per > 1:  # the last sequence shares the first page of the first
            k = int((table[-1] >= 0).sum())
            table[-1, k] = table[0, 0]
            refs[table[0, 0]] += 1
        st.update(pages=c["pages"], max_pages=table.shape[1], table=_i32(table), refs=_i32(refs),
                  new_table=torch.empty(table.shape, dtype=torch.int32, device=DEV),
                  new_refs=torch.empty(c["pages"], dtype=torch.int32, device=DEV),
                  used=torch.empty(1, dtype=torch.int32, device=DEV))
    elif c["op"] == "fork":
        lens = _lens(c)
        need = lens // c["page"] + 1  # the last page has room
        pages = int(need.sum()) + c["spare"]
        max_pages = int(need.max()) + 1 + -(-c["reserve"] // c["page"])
        table = _table(rng, need, max_pages, pages)
        refs = np.zeros(pages, np.int32)
        refs[table[table >= 0]] = 1
        st.update(pages=pages, max_pages=max_pages, table=_i32(table), refs=_i32(refs), lens=_i32(lens), parent=_i32(_parents(c, rng)),
                  new_table=torch.empty(table.shape, dtype=torch.int32, device=DEV),
                  new_refs=torch.empty(pages, dtype=torch.int32, device=DEV),
                  new_lens=torch.empty(c["B"], dtype=torch.int32, device=DEV), short=torch.empty(1, dtype=torch.int32, device=DEV))
    else:
        old = rng.integers(0, 40, c["B"]) if c["op"] == "append" else _lens(c)  # rows before this pass
        new = _lens(c) if c["op"] == "append" else _nodes(c)
        lens = old + new
        need = -(-lens // c["page"])
        pages, max_pages = int(need.sum()) + 3, max(1, int(need.max()))
        st.update(pages=pages, max_pages=max_pages, table=_i32(_table(rng, need, max_pages, pages)), pos=_i32(old), lens=_i32(lens),
                  nodes=_i32(new))
        if c["op"] != "tree":
            # the tokens' K and V as the slices of one projection's output they are
            heads = 2 * c["Hkv"] + 1
            tokens = int(new.sum())
            x = torch.randn(tokens, heads, c["D"], generator=gen, device=DEV).to(DTYPE[c["in"]])
            st.update(k=x[:, 1:1 + c["Hkv"]], v=x[:, 1 + c["Hkv"]:], cu=_i32(np.concatenate([[0], np.cumsum(new)])))
        if c["op"] != "append":
            B, Q = c["B"], c["Q"]
            parent = (rng.random((B, Q)) * (np.arange(Q) + 1)).astype(np.int64) - 1  # -1: a child of the last row
            parent = np.where(rng.random((B, Q)) < 0.5, np.arange(Q) - 1, parent)  # half of them go on from the one before
            mask = np.zeros((B, Q), np.uint64)
            for i in range(Q):
                up = np.where(parent[:, i] < 0, np.uint64(0), mask[np.arange(B), np.maximum(parent[:, i], 0)])
                mask[:, i] = up | np.uint64(1 << i)
            st.update(mask=torch.from_numpy(mask.view(np.int64)).to(DEV),
                      q=torch.randn(B, Q, c["Hq"], c["D"], generator=gen, device=DEV).half(),
                      out=torch.empty(B, Q, c["Hq"], c["D"], dtype=torch.float16, device=DEV))
            if c["op"] == "step":  # the accepted path: from the root to one of the nodes
                leaf = (rng.random(B) * new).astype(np.int64)
                path = np.full((B, Q), -1, np.int32)
                for b in range(B):
                    ids = [i for i in range(Q) if int(mask[b, leaf[b]]) >> i & 1]
                    path[b, :len(ids)] = ids
                st.update(path=_i32(path), accepted=_i32((path >= 0).sum(1)), new_lens=torch.empty(B, dtype=torch.int32, device=DEV))
    st["K"], st["scK"] = _fill(c, gen, st["pages"], True)
    st["V"], st["scV"] = _fill(c, gen, st["pages"], False)
    return st


# ---- one pass -------------------------------------------------------------------------------


def run(state):
    return (_run_own if own else _run_plain)(state)


def _pool(st):
    """The cache as run() returns it: 16-bit and fp8 rows as their numbers, integer codes as whole numbers (a byte of
    packed ones is the same exactly when all its codes are)."""
    see = {"f16+": torch.float16, "bf16+": torch.bfloat16, "f8+": torch.float8_e4m3fn, "q8+": torch.int8}.get(st["case"]["fmt"], torch.uint8)
    d = {"K": st["K"].view(see), "V": st["V"].view(see)}
    if st["scK"] is not None:
        d.update(scK=st["scK"], scV=st["scV"])
    return d


def _run_own(st):
    import voltattn_b200 as va

    c = st["case"]
    fmt, B, Hkv, D, page, pages, mp = c["fmt"], c["B"], c["Hkv"], c["D"], c["page"], st["pages"], st["max_pages"]
    b = va.DeviceBufs(st["K"], st["V"], st["scK"], st["scV"], st.get("q"), st.get("out"), st["ws"])
    if c["op"] == "compact":
        va.compact_pages(fmt, b, st["refs"], st["table"], st["new_refs"], st["new_table"], st["used"], B, mp, Hkv, page, pages, D,
                         layers=c["layers"])
        return {**_pool(st), "refs": st["new_refs"], "table": st["new_table"], "used": st["used"]}
    if c["op"] == "fork":
        va.fork_pages(fmt, b, st["refs"], st["table"], st["lens"], st["parent"], st["new_refs"], st["new_table"], st["new_lens"],
                      st["short"], B, B, mp, c["reserve"], Hkv, page, pages, D, layers=c["layers"])
        return {**_pool(st), "refs": st["new_refs"], "table": st["new_table"], "lens": st["new_lens"], "short": st["short"]}
    if c["op"] in ("append", "step"):
        va.append_packed(fmt, st["k"], st["v"], b, st["table"], mp, st["cu"], st["pos"], B, Hkv, page, pages, D)
        if c["op"] == "append":
            return _pool(st)
    va.decode_tree(fmt, b, st["mask"], st["lens"], st["nodes"], st["table"], mp, B, c["Hq"], Hkv, c["Q"], page, pages, D)
    if c["op"] == "tree":
        return {"out": st["out"]}
    va.accept_tree(fmt, b, st["table"], mp, st["lens"], st["nodes"], st["path"], st["accepted"], st["new_lens"], B, c["Q"], Hkv, page,
                   pages, D)
    return {**_pool(st), "out": st["out"], "lens": st["new_lens"]}


def _values(codes, scales, fmt):
    """fp32 values of rows of codes [..., bytes]."""
    if fmt == "f16+":
        return codes.view(torch.float16).float()
    if fmt == "bf16+":
        return codes.view(torch.bfloat16).float()
    if fmt == "f8+":
        v = codes.view(torch.float8_e4m3fn).float()
    elif fmt == "q8+":
        v = codes.view(torch.int8).float()
    elif fmt == "q4+":
        v = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float() - 8
    else:
        t = codes.reshape(*codes.shape[:-1], -1, 3).int()
        w = (t[..., 0] | t[..., 1] << 8 | t[..., 2] << 16).unsqueeze(-1)
        v = (w >> torch.arange(0, 24, 3, device=codes.device) & 7).flatten(-2).float() - 4
    return (v.unflatten(-1, (-1, 64)) * scales.float().unsqueeze(-1)).flatten(-2)


def _plain_tree(st):
    c = st["case"]
    B, Hq, Hkv, Q, D, page = c["B"], c["Hq"], c["Hkv"], c["Q"], c["D"], c["page"]
    L, G = st["max_pages"] * page, Hq // Hkv
    t = st["table"].clamp(min=0).long()

    def side(codes, scales):  # [B, Hkv, L, D]
        own_pages = codes.view(st["pages"], Hkv, page, -1)[t]
        x = _values(own_pages, None if scales is None else scales.view(st["pages"], Hkv, page, -1)[t], c["fmt"])
        return x.transpose(1, 2).reshape(B, Hkv, L, D)

    n, ctx = st["nodes"].long(), (st["lens"] - st["nodes"]).long()
    j = torch.arange(L, device=DEV)[None, :] - ctx[:, None]  # the drafted token of each row; < 0: before them
    drafted = (st["mask"][:, :, None] >> j.clamp(0, 63)[:, None, :] & 1).bool() & ((j >= 0) & (j < n[:, None]))[:, None, :]
    vis = (drafted | (j < 0)[:, None, :]) & (torch.arange(Q, device=DEV)[None, :] < n[:, None])[:, :, None]  # [B, Q, L]
    q = st["q"].float().view(B, Q, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * Q, D)
    s = (q @ side(st["K"], st["scK"]).transpose(-1, -2)).mul_(1.0 / D ** 0.5).view(B, Hkv, G, Q, L)
    s = s.masked_fill_(~vis[:, None, None], float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(m > float("-inf"), m, torch.zeros_like(m))).exp_()
    l = p.sum(-1, keepdim=True)
    o = (p.view(B, Hkv, G * Q, L) @ side(st["V"], st["scV"])).view(B, Hkv, G, Q, D)
    o = torch.where(l > 0, o / l, torch.zeros_like(o))
    return o.permute(0, 3, 1, 2, 4).reshape(B, Q, Hq, D).half()


def _plain_append(st):
    c = st["case"]
    page, Hkv = c["page"], c["Hkv"]
    T = st["k"].shape[0]
    i = torch.arange(T, device=DEV)
    b = torch.searchsorted(st["cu"][1:].long(), i, right=True)
    p = st["pos"].long()[b] + i - st["cu"].long()[b]
    row = (st["table"].long()[b, p // page] * Hkv)[:, None] + torch.arange(Hkv, device=DEV)
    row = row * page + (p % page)[:, None]
    for x, codes, scales in ((st["k"], st["K"], st["scK"]), (st["v"], st["V"], st["scV"])):
        k, s = _quantize(x, c["fmt"])
        codes[row] = k
        if s is not None:
            scales[row] = s


def _plain_accept(st):
    c = st["case"]
    page, Hkv, P = c["page"], c["Hkv"], c["Q"]
    ctx = (st["lens"] - st["nodes"]).long()
    i = torch.arange(P, device=DEV)[None, :]
    ok = (i < st["accepted"][:, None]).flatten()
    b = torch.arange(c["B"], device=DEV)[:, None].expand(-1, P).flatten()[ok]

    def rows(p):
        r = (st["table"].long()[b, p // page] * Hkv)[:, None] + torch.arange(Hkv, device=DEV)
        return r * page + (p % page)[:, None]

    src = rows((ctx[:, None] + st["path"].clamp(min=0)).flatten()[ok])
    dst = rows((ctx[:, None] + i).flatten()[ok])
    for x in (st["K"], st["V"], st["scK"], st["scV"]):
        if x is not None:
            x[dst] = x[src]
    torch.add(ctx, st["accepted"], out=st["new_lens"])


def _plain_fork(st):
    c = st["case"]
    B, mp, page = c["B"], st["max_pages"], c["page"]
    table, refs, lens, par = st["table"].long(), st["refs"], st["lens"].long(), st["parent"].long()
    i = torch.arange(B, device=DEV)
    has = par >= 0
    src = par.clamp(min=0)
    kids = torch.zeros(B, dtype=torch.long, device=DEV).index_add_(0, src, has.long())
    first = torch.full((B,), B, device=DEV).scatter_reduce_(0, src, torch.where(has, i, B), "amin")
    keeps = has & (first[src] == i)  # the first to go on keeps the sequence's own pages
    j = torch.arange(mp, device=DEV)[None, :]
    full = lens // page
    new_lens = torch.where(has, lens[src], torch.zeros_like(src))
    held = torch.where(keeps[:, None], table[src], torch.where(has[:, None] & (j < full[src][:, None]), table[src], -1))
    need = torch.where(has, (new_lens + c["reserve"] + page - 1) // page, torch.zeros_like(src)).clamp(max=mp)
    ask = (held < 0) & (j < need[:, None])
    rank = ask.flatten().long().cumsum(0).view(B, mp) - 1
    free = torch.nonzero(refs == 0).flatten()
    n = free.numel()
    given = ask & (rank < n)
    held = torch.where(given, free[rank.clamp(0, max(n - 1, 0))] if n else held, held)
    short = (ask & ~given).sum()
    # a sequence that got no page for its last rows ends before them
    part = new_lens // page
    lost = (ask & ~given & (j == part[:, None]) & (new_lens % page > 0)[:, None]).any(1)
    new_lens = torch.where(lost, part * page, new_lens)
    copied = given & (j == part[:, None]) & (new_lens % page > 0)[:, None] & ~keeps[:, None]
    delta = torch.where(j < full[:, None], (kids - 1)[:, None], torch.where(kids > 0, 0, -1)[:, None])
    delta = torch.where(table >= 0, delta, torch.zeros_like(delta))
    st["new_refs"].copy_(refs)
    st["new_refs"].index_add_(0, table.clamp(min=0).flatten(), delta.flatten().int())
    st["new_refs"].index_add_(0, held.clamp(min=0).flatten(), given.flatten().int())
    st["new_table"].copy_(held)
    st["new_lens"].copy_(new_lens)
    st["short"].copy_(short.view(1))
    # the rows of the last page, in whole blocks of eight
    k = copied.any(1)
    to, frm = held.gather(1, part[:, None].clamp(max=mp - 1))[k, 0], table[src].gather(1, part[:, None].clamp(max=mp - 1))[k, 0]
    n_rows = (new_lens[k] % page + 7) // 8 * 8
    for x in (st["K"], st["V"], st["scK"], st["scV"]):
        if x is not None:
            y = x.view(c["layers"], st["pages"], c["Hkv"], page, -1)
            take = (torch.arange(page, device=DEV)[None, :] < n_rows[:, None])[None, :, None, :, None]
            y[:, to] = torch.where(take, y[:, frm], y[:, to])


def _plain_compact(st):
    c = st["case"]
    refs, table = st["refs"], st["table"].long()
    used = refs > 0
    n = used.sum()
    at = torch.arange(c["pages"], device=DEV)
    move, hole = used & (at >= n), ~used & (at < n)
    src, dst = torch.nonzero(move).flatten(), torch.nonzero(hole).flatten()
    to = at.clone()
    to[src] = dst
    for x in (st["K"], st["V"], st["scK"], st["scV"]):
        if x is not None:
            y = x.view(c["layers"], st["pages"], -1)
            y[:, dst] = y[:, src]
    st["new_refs"].copy_(torch.where(at < n, refs, torch.zeros_like(refs)))
    st["new_refs"][dst] = refs[src]
    st["new_table"].copy_(torch.where(table >= 0, to[table.clamp(min=0)], table))
    st["used"].copy_(n.view(1))


def _run_plain(st):
    op = st["case"]["op"]
    if op == "tree":
        return {"out": _plain_tree(st)}
    if op == "compact":
        _plain_compact(st)
        return {**_pool(st), "refs": st["new_refs"], "table": st["new_table"], "used": st["used"]}
    if op == "fork":
        _plain_fork(st)
        return {**_pool(st), "refs": st["new_refs"], "table": st["new_table"], "lens": st["new_lens"], "short": st["short"]}
    _plain_append(st)
    if op == "append":
        return _pool(st)
    out = _plain_tree(st)
    _plain_accept(st)
    return {**_pool(st), "out": out, "lens": st["new_lens"]}


# ---- the same in 64 bits --------------------------------------------------------------------


def _exact_rows(codes, scales, fmt):
    """float64 values of rows of codes (numpy bytes [n, bytes])."""
    n = codes.shape[0]
    if fmt == "f16+":
        return codes.view(np.float16).astype(np.float64)
    if fmt == "bf16+":
        return (codes.view(np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    if fmt == "f8+":
        e, m = (codes >> 3 & 15).astype(np.int64), (codes & 7).astype(np.float64)
        v = np.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * 2.0 ** (e - 7.0)) * np.where(codes & 128, -1.0, 1.0)
    elif fmt == "q8+":
        v = codes.view(np.int8).astype(np.float64)
    else:
        bits = np.unpackbits(codes, axis=1, bitorder="little").reshape(n, -1, BITS[fmt]).astype(np.float64)
        v = bits @ (2.0 ** np.arange(BITS[fmt])) - 2.0 ** (BITS[fmt] - 1)
    return v * np.repeat(scales.astype(np.float64), 64, axis=1)


def exact(case, seed):
    """The attention outputs in 64 bits; what is whole numbers or copied has no such value. None where it would be slow."""
    c = case
    if c["op"] not in ("tree", "step") or work(c)["flops"] > 4e11:
        return None
    st = prepare(c, seed)
    B, Hkv, D, Q, page = c["B"], c["Hkv"], c["D"], c["Q"], c["page"]
    G = c["Hq"] // Hkv
    if c["op"] == "step":
        _plain_append(st)  # quantized codes: whole numbers, the same by definition
    out = torch.zeros(B, Q, c["Hq"], D, dtype=torch.float64, device=DEV)
    table, lens, nodes, mask = (st[k].cpu().numpy() for k in ("table", "lens", "nodes", "mask"))
    byte = [st[k].view(st["pages"], Hkv, page, -1) if st[k] is not None else None for k in ("K", "scK", "V", "scV")]
    for b in range(B):
        L, n = int(lens[b]), int(nodes[b])
        ids = torch.from_numpy(table[b, :-(-L // page)].astype(np.int64)).to(DEV)
        see = torch.ones(n, L, dtype=torch.bool)
        see[:, L - n:] = torch.from_numpy(mask[b, :n].astype(np.uint64)[:, None] >> np.arange(n, dtype=np.uint64)[None, :] & np.uint64(1) != 0)
        see = see.to(DEV).repeat(G, 1)
        for h in range(Hkv):
            side = []
            for k in (0, 2):
                cs = byte[k][ids, h].reshape(-1, byte[k].shape[-1])[:L].cpu().numpy()
                sc = byte[k + 1][ids, h].reshape(-1, byte[k + 1].shape[-1])[:L].cpu().numpy() if byte[k + 1] is not None else None
                side.append(torch.from_numpy(np.ascontiguousarray(_exact_rows(cs, sc, c["fmt"]))).to(DEV))
            q = st["q"][b, :n, h * G:(h + 1) * G].double().transpose(0, 1).reshape(G * n, D)
            s = (q @ side[0].T / np.sqrt(float(D))).masked_fill(~see, float("-inf"))
            o = torch.softmax(s, -1) @ side[1] if L else torch.zeros(G * n, D, dtype=torch.float64, device=DEV)
            out[b, :n, h * G:(h + 1) * G] = o.view(G, n, D).transpose(0, 1)
    return {"out": out}
