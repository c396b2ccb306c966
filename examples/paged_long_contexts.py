"""Serving many questions about one long document: heads normed and positions of three axes, the document's attention
weights gathered while it is read, its cache cut to the rows that matter, and the rest shared by everybody who asks.

A small model with random fp16 weights (that of paged_serving.py, its queries and keys normed head by head):

  read    the document in chunks; `paged.weighted_attention` sums up what every row was worth, for each layer and kv head;
  cut     `paged.evict` keeps the first and the last rows and the heaviest of the others, in fresh pages;
  answer  the users' questions and answers behind the document's pages, which all of them share:
          `paged.shared_attention` reads them once for a step of the whole batch.

Run from the repository's root:  python examples/paged_long_contexts.py
"""

import os
import sys

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

import torch

from paged_serving import Cache, Model, ints, starts

import paged
import qmm


class LongModel(Model):
    """`forward` takes positions [3, tokens] (time, height, width) and a call that attends for a layer."""

    def __init__(self, seed=0, **kw):
        super().__init__(seed=seed, **kw)
        g = torch.Generator(device="cuda").manual_seed(seed + 1)
        self.q_norm, self.k_norm = (1 + 0.1 * torch.randn(2, self.head_dim, generator=g, device="cuda")).half()
        half = self.head_dim // 2
        self.axes = [0] * (half // 4) + [1] * (half * 3 // 8) + [2] * (half - half // 4 - half * 3 // 8)

    def forward(self, tokens, cache, table, cu, ctx, positions, attend):
        x = self.embed[tokens]
        H, K, D = self.heads, self.kv_heads, self.head_dim
        for i, b in enumerate(self.blocks):
            qkv = self._mm(self._norm(x), b["qkv"]).view(-1, H + 2 * K, D)
            q = paged.append(qkv[:, H:H + K], qkv[:, H + K:], cache.k[i], cache.v[i], table, cu, ctx, q=qkv[:, :H], positions=positions,
                             neox=True, q_norm=self.q_norm, k_norm=self.k_norm, axes=self.axes)
            x = x + self._mm(attend(i, q).view(-1, H * D), b["o"])
            h = self._norm(x)
            gate, up = self._mm(h, b["gate"]), self._mm(h, b["up"])
            act = torch.empty_like(gate)
            qmm.check(qmm.lib().qmm_swiglu(gate.data_ptr(), up.data_ptr(), act.data_ptr(), act.numel(), qmm._stream_handle()))
            x = x + self._mm(act, b["down"])
        return qmm.gemm(qmm.GGML_F16, self._norm(x), self.head, self.vocab, self.hidden)


def text_positions(first, count):
    """A text's tokens are at the same place on every axis."""
    return [list(range(first, first + count))] * 3


def picture_positions(first, rows, columns):
    """The patches of a picture: one time, their row and their column."""
    return [[first] * (rows * columns), [first + i // columns for i in range(rows * columns)], [first + i % columns for i in range(rows * columns)]]


def joined(*parts):
    return [sum((p[a] for p in parts), []) for a in range(3)]


def read(model, cache, document, positions, chunk=32):
    """Runs the document; (its pages, the sums of its rows' attention weights [layers, 1, kv_heads, rows])."""
    pages, n = [], 0
    weights = torch.zeros(model.layers, 1, model.kv_heads, -(-len(document) // cache.page_size) * cache.page_size, device="cuda")
    while n < len(document):
        part = document[n:n + chunk]
        table = cache.grow([pages], [n + len(part)])
        cu, ctx = ints([0, len(part)]), ints([n])

        def attend(i, q):
            return paged.weighted_attention(q, cache.k[i], cache.v[i], table, cu, ctx, weights[i], max_new=len(part))[0]

        model.forward(torch.tensor(part, device="cuda"), cache, table, cu, ctx, ints([p[n:n + len(part)] for p in positions]), attend)
        n += len(part)
    return pages, weights


def cut(cache, pages, rows, weights, keep, recent=16, sinks=4):
    """The pages and the length of the document once its cache holds at most `keep` rows, and their weights."""
    fresh = [cache.free.pop() for _ in range(-(-keep // cache.page_size))]
    table, lens, weights = paged.evict(cache.k, cache.v, ints([pages]), ints([rows]), weights, ints([fresh]), keep, recent=recent, sinks=sinks)
    kept = [p for p in table[0].tolist() if p >= 0]
    cache.free += [p for p in pages + fresh if p not in kept]
    return kept, lens.item(), weights


def answer(model, cache, pages, rows, position, questions, steps, share=True):
    """Greedy answers to questions about a document of `rows` cached rows; (tokens, the first step's logits).  A user's own rows
    begin in a page of their own, into which the document's open page is copied."""
    full = rows // cache.page_size
    tables, ctx = [pages[:full] for _ in questions], [rows] * len(questions)
    for t in tables if rows % cache.page_size else []:
        t.append(cache.free.pop())
        cache.k[:, t[-1]], cache.v[:, t[-1]] = cache.k[:, pages[full]], cache.v[:, pages[full]]
    groups, shared = ints([0, len(questions)]), ints([full * cache.page_size])
    place, tokens, out, first = [position] * len(questions), questions, [[] for _ in questions], None
    for _ in range(steps):
        counts = [len(t) for t in tokens]
        table = cache.grow(tables, [c + n for c, n in zip(ctx, counts)])
        cu, lens, most = ints(starts(counts)), ints(ctx), max(counts)

        def attend(i, q):
            if share:
                return paged.shared_attention(q, cache.k[i], cache.v[i], table, cu, lens, groups, shared, max_new=most)
            return paged.tree_attention(q, cache.k[i], cache.v[i], table, cu, lens, max_new=most)

        at = joined(*(text_positions(p, n) for p, n in zip(place, counts)))
        logits = model.forward(torch.tensor(sum(tokens, []), device="cuda"), cache, table, cu, lens, ints(at), attend)
        last = logits[[c - 1 for c in starts(counts)[1:]]]
        first = last if first is None else first
        ctx, place = [c + n for c, n in zip(ctx, counts)], [p + n for p, n in zip(place, counts)]
        tokens = [[t] for t in last.argmax(-1).tolist()]
        for o, t in zip(out, tokens):
            o += t
    return out, first


def make(model, seed=1):
    """A document of text, a picture and text, with its positions, and questions of several lengths."""
    g = torch.Generator().manual_seed(seed)
    words = lambda n: torch.randint(model.vocab, (n,), generator=g).tolist()  # noqa: E731
    positions = joined(text_positions(0, 50), picture_positions(50, 6, 9), text_positions(59, 61))
    return words(50 + 54 + 61), positions, [words(n) for n in (3, 7, 1, 5)]


def main():
    model = LongModel()
    document, positions, questions = make(model)
    cache = Cache(model, 96)
    pages, weights = read(model, cache, document, positions)
    end = positions[0][-1] + 1
    whole, _ = answer(model, cache, pages, len(document), end, questions, 8)
    pages, rows, _ = cut(cache, pages, len(document), weights, keep=80)
    print(f"the document's {len(document)} rows are cut to {rows}")
    for a, b in zip(whole, answer(model, cache, pages, rows, end, questions, 8)[0]):
        print(f"of all rows {a}, of those kept {b}")


if __name__ == "__main__":
    main()
