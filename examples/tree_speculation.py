"""Speculative decoding with a tree over a paged 4-bit cache, end to end.

A toy language model (an embedding, one attention layer with grouped heads, a
vocabulary projection; random weights) answers a few prompts greedily, twice:
one token at a time, and with trees of drafted tokens. Both give the same tokens.
The second is the loop of a serving engine around this package's operators:

    append_packed   the prompts', then the drafted tokens' K and V into their pages
    fork_pages      a page for every sequence's next rows (and copies of a sequence)
    decode_tree     all drafted tokens of all sequences in one call
    accept_tree     the accepted path's rows moved together
    compact_pages   the pages in use moved to the front when requests have ended

    python examples/tree_speculation.py [--tokens 24] [--device cuda:0]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import voltattn_b200 as va  # noqa: E402

FMT, HQ, HKV, D, PAGE, VOCAB = "q4+", 8, 2, 128, 32, 61


class ToyModel:
    """logits(x) = Attention(x Wq, cache of x Wk, x Wv) Wo, x = embedding + position."""

    def __init__(self, device, seed=0):
        g = torch.Generator(device=device).manual_seed(seed)
        n = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
        self.embed, self.place = n(VOCAB, 64), n(4096, 64) * 0.5
        self.wq, self.wk, self.wv = n(64, HQ * D) / 8, n(64, HKV * D) / 8, n(64, HKV * D) / 8
        self.wo, self.skip = n(HQ * D, VOCAB) / 8, n(64, VOCAB) / 2

    def inputs(self, tokens, places):
        """x, q [..., HQ, D] and k, v [..., HKV, D] of tokens at their places."""
        x = self.embed[tokens] + self.place[places]
        heads = lambda w, n: (x @ w).half().view(*tokens.shape, n, D)  # noqa: E731
        return x, heads(self.wq, HQ), heads(self.wk, HKV), heads(self.wv, HKV)

    def next_tokens(self, x, attended):
        return (attended.float().flatten(-2) @ self.wo + x @ self.skip).argmax(-1)


class Cache:
    """A page pool with the tables of B sequences, grown and reordered by fork_pages."""

    def __init__(self, B, pages, max_pages, device):
        self.B, self.pages, self.max_pages = B, pages, max_pages
        z = lambda *s: torch.zeros(*s, dtype=torch.int32, device=device)  # noqa: E731
        rows = pages * HKV * PAGE
        self.K, self.V = (torch.zeros(rows, va.payload_bytes(FMT, D), dtype=torch.uint8, device=device) for _ in "KV")
        self.sK, self.sV = (torch.zeros(rows, D // 64, dtype=torch.float16, device=device) for _ in "KV")
        self.refs, self.table, self.lens = z(pages), torch.full((B, max_pages), -1, dtype=torch.int32, device=device), z(B)
        self.short, self.used = z(1), z(1)
        self.ws = torch.zeros(va.tree_workspace_bytes(B, HQ, HKV, 64, D, 16), dtype=torch.uint8, device=device)
        self.scratch = torch.zeros(va.pages_workspace_bytes(B, max_pages, pages), dtype=torch.uint8, device=device)

    def bufs(self, q=None, out=None, ws=None):
        return va.DeviceBufs(self.K, self.V, self.sK, self.sV, q, out, self.ws if ws is None else ws)

    def reorder(self, parent, reserve):
        """New sequence i continues parent[i] (-1: ends), with pages for `reserve` more rows."""
        refs, table, lens = torch.empty_like(self.refs), torch.empty_like(self.table), torch.empty_like(self.lens)
        va.fork_pages(FMT, self.bufs(ws=self.scratch), self.refs, self.table, self.lens, parent, refs, table, lens,
                      self.short, self.B, self.B, self.max_pages, reserve, HKV, PAGE, self.pages, D)
        self.refs, self.table, self.lens = refs, table, lens

    def append(self, k, v, counts):
        """Rows of packed tokens after each sequence's last; counts int32 [B]."""
        cu = torch.nn.functional.pad(counts.cumsum(0), (1, 0)).int()
        va.append_packed(FMT, k, v, self.bufs(), self.table, self.max_pages, cu, self.lens, self.B, HKV, PAGE, self.pages, D)
        self.lens = self.lens + counts

    def attend(self, q, mask, nodes):
        """q [B][Q][HQ][D] of the drafted tokens, the last nodes[b] rows of each sequence."""
        out = torch.empty_like(q)
        va.decode_tree(FMT, self.bufs(q, out), mask, self.lens, nodes, self.table, self.max_pages, self.B, HQ, HKV,
                       q.shape[1], PAGE, self.pages, D)
        return out

    def accept(self, nodes, path, accepted):
        lens = torch.empty_like(self.lens)
        va.accept_tree(FMT, self.bufs(), self.table, self.max_pages, self.lens, nodes, path, accepted, lens, self.B,
                       path.shape[1], HKV, PAGE, self.pages, D)
        self.lens = lens

    def compact(self):
        refs, table = torch.empty_like(self.refs), torch.empty_like(self.table)
        va.compact_pages(FMT, self.bufs(ws=self.scratch), self.refs, self.table, refs, table, self.used, self.B,
                         self.max_pages, HKV, PAGE, self.pages, D)
        self.refs, self.table = refs, table
        return int(self.used)


def prefill(model, cache, prompts, device):
    """All but the prompts' last tokens into the cache; the last ones start the decoding."""
    B = len(prompts)
    cache.reorder(torch.arange(B, dtype=torch.int32, device=device), max(map(len, prompts)))
    packed = torch.cat([torch.tensor(p[:-1], dtype=torch.long, device=device) for p in prompts])
    places = torch.cat([torch.arange(len(p) - 1, device=device) for p in prompts])
    _, _, k, v = model.inputs(packed, places)
    cache.append(k, v, torch.tensor([len(p) - 1 for p in prompts], dtype=torch.int32, device=device))
    return torch.tensor([p[-1] for p in prompts], device=device)


# The tree: node 0 is the last accepted token; every other node drafts what follows its parent.
PARENT = [-1, 0, 0, 0, 1, 1, 2, 4, 4, 7]
DEPTH = [0, 1, 1, 1, 2, 2, 2, 3, 3, 4]


def tree_masks():
    masks = []
    for i, p in enumerate(PARENT):
        masks.append((masks[p] if p >= 0 else 0) | 1 << i)
    return masks


def decode(model, prompts, tokens, device, drafts=None):
    """`tokens` greedy tokens for each prompt. drafts: the answers that the drafting guesses from
    (None: one token at a time). Returns them, the number of steps and the cache."""
    B, Q = len(prompts), len(PARENT) if drafts is not None else 1
    most = max(map(len, prompts)) + tokens + 2 * Q
    cache = Cache(B, B * (most // PAGE + 2), most // PAGE + 2, device)
    last = prefill(model, cache, prompts, device)
    mask = torch.tensor(tree_masks()[:Q], device=device).expand(B, Q).contiguous()
    nodes = torch.full((B,), Q, dtype=torch.int32, device=device)
    depth = torch.tensor(DEPTH[:Q], device=device)
    same = torch.arange(B, dtype=torch.int32, device=device)
    gen = torch.Generator().manual_seed(1)
    answers, steps = [[] for _ in range(B)], 0
    while min(map(len, answers)) < tokens:
        steps += 1
        cache.reorder(same, Q)
        draft = torch.randint(VOCAB, (B, Q), generator=gen)
        if drafts is not None:  # a drafting model that is often right
            for b in range(B):
                for i in range(1, Q):
                    at = len(answers[b]) + DEPTH[i] - 1
                    if at < tokens and torch.rand((), generator=gen) < 0.7:
                        draft[b, i] = drafts[b][at]
        draft = draft.to(device)
        draft[:, 0] = last
        x, q, k, v = model.inputs(draft, cache.lens[:, None] + depth)
        cache.append(k.flatten(0, 1), v.flatten(0, 1), nodes)
        follows = model.next_tokens(x, cache.attend(q, mask, nodes)).tolist()  # after each node
        drafted, path = draft.tolist(), torch.zeros(B, Q, dtype=torch.int32)
        accepted, fresh = [], []
        for b in range(B):
            node, walk = 0, [0]
            while True:
                answers[b].append(follows[b][node])
                child = [i for i in range(node + 1, Q) if PARENT[i] == node and drafted[b][i] == follows[b][node]]
                if not child:
                    break
                node = child[0]
                walk.append(node)
            path[b, :len(walk)] = torch.tensor(walk)
            accepted.append(len(walk))
            fresh.append(answers[b][-1])
        cache.accept(nodes, path.to(device), torch.tensor(accepted, dtype=torch.int32, device=device))
        last = torch.tensor(fresh, device=device)
    return [a[:tokens] for a in answers], steps, cache


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--tokens", type=int, default=24)
    ap.add_argument("--device", default="cuda:0")
    a = ap.parse_args(argv)
    gen = torch.Generator().manual_seed(3)
    prompts = [torch.randint(VOCAB, (n,), generator=gen).tolist() for n in (5, 70, 33, 128)]
    with torch.cuda.device(a.device):
        model = ToyModel(a.device)
        plain, n1, _ = decode(model, prompts, a.tokens, a.device)
        tree, n2, cache = decode(model, prompts, a.tokens, a.device, drafts=plain)
        print(f"{a.tokens} tokens for {len(prompts)} prompts: {n1} steps one by one, {n2} with trees of {len(PARENT)}")
        assert tree == plain, "the trees' tokens differ from the ones decoded one by one"
        # two requests end, a third is sampled twice from here on; the pool shrinks to its used pages
        keep = torch.tensor([1, 1, 3, -1], dtype=torch.int32, device=a.device)
        cache.reorder(keep, 1)
        print(f"after the fork: lengths {cache.lens.tolist()}, {cache.compact()} of {cache.pages} pages in use")
        assert va.device_error() == 0
    return n1, n2


if __name__ == "__main__":
    main()
