"""Serving with a paged cache: chunked prompts, drafted trees, beam search.

A small Llama-shaped model with random fp16 weights, run with the framework's calls: projections by `qmm.gemm`, norms and
SwiGLU by the C ABI, the cache by `paged` and `beam`.  Three ways to continue a batch of prompts:

  greedy       one token a step (the plain form of decoding);
  speculative  a drafted tree a step: its nodes attend to their ancestors (`paged.tree_attention`), the longest path that
               the model agrees with is kept (`paged.commit_path`);
  beams        the best of several hypotheses (`beam.select`, `beam.reorder`).

Run from the repository's root:  python examples/paged_serving.py
"""

import os
import sys

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gfx1150-inference_amd"))

import torch

import beam
import paged
import qmm


class Model:
    """Random weights; `forward` runs new tokens of a batch of sequences against the cache and returns their logits."""

    def __init__(self, layers=2, hidden=256, heads=8, kv_heads=2, head_dim=64, inner=512, vocab=512, seed=0):
        self.layers, self.hidden, self.heads, self.kv_heads, self.head_dim, self.inner, self.vocab = layers, hidden, heads, kv_heads, head_dim, inner, vocab
        g = torch.Generator(device="cuda").manual_seed(seed)
        mat = lambda n, k: (torch.randn(n, k, generator=g, device="cuda") / k ** 0.5).half()  # noqa: E731
        self.embed = torch.randn(vocab, hidden, generator=g, device="cuda").half()
        self.head = mat(vocab, hidden) * 3
        self.norm = torch.ones(hidden, dtype=torch.float16, device="cuda")
        self.blocks = [dict(qkv=mat((heads + 2 * kv_heads) * head_dim, hidden), o=mat(hidden, heads * head_dim), gate=mat(inner, hidden),
                            up=mat(inner, hidden), down=mat(hidden, inner)) for _ in range(layers)]

    def _norm(self, x):
        out = torch.empty_like(x)
        qmm.check(qmm.lib().qmm_rmsnorm(x.data_ptr(), self.norm.data_ptr(), qmm.DTYPE_F16, out.data_ptr(), x.shape[0], self.hidden, 1e-5,
                                        qmm._stream_handle()))
        return out

    def _mm(self, x, w):
        return qmm.gemm(qmm.GGML_F16, x, w, w.shape[0], w.shape[1], out_dtype=torch.float16)

    def forward(self, tokens, cache, table, cu, ctx, positions=None, mask=None, max_new=None):
        x = self.embed[tokens]
        H, K, D = self.heads, self.kv_heads, self.head_dim
        for i, b in enumerate(self.blocks):
            qkv = self._mm(self._norm(x), b["qkv"]).view(-1, H + 2 * K, D)
            # the rotation is on the way into the cache; the slices of the fused projection are taken as they lie
            q = paged.append(qkv[:, H:H + K], qkv[:, H + K:], cache.k[i], cache.v[i], table, cu, ctx, q=qkv[:, :H], positions=positions)
            a = paged.tree_attention(q, cache.k[i], cache.v[i], table, cu, ctx, mask=mask, max_new=max_new)
            x = x + self._mm(a.view(-1, H * D), b["o"])
            h = self._norm(x)
            gate, up = self._mm(h, b["gate"]), self._mm(h, b["up"])
            act = torch.empty_like(gate)
            qmm.check(qmm.lib().qmm_swiglu(gate.data_ptr(), up.data_ptr(), act.data_ptr(), act.numel(), qmm._stream_handle()))
            x = x + self._mm(act, b["down"])
        return qmm.gemm(qmm.GGML_F16, self._norm(x), self.head, self.vocab, self.hidden)


class Cache:
    """Pages for every layer, and a free list that the host keeps."""

    def __init__(self, model, pages, page_size=16):
        shape = (model.layers, pages, model.kv_heads, page_size, model.head_dim)
        self.k, self.v = (torch.empty(shape, dtype=torch.float16, device="cuda") for _ in range(2))
        self.page_size, self.free = page_size, list(range(pages - 1, -1, -1))

    def grow(self, tables, lengths):
        """Pages so that sequence b can hold lengths[b] rows; the tables as a tensor."""
        for row, n in zip(tables, lengths):
            while len(row) * self.page_size < n:
                row.append(self.free.pop())
        width = max(map(len, tables))
        return ints([row + [-1] * (width - len(row)) for row in tables])


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def pages_of(table):
    return {p for row in table.tolist() for p in row if p >= 0}


def starts(counts):
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    return cu


def prefill(model, cache, prompts, chunk=24):
    """Runs the prompts in chunks; (tables, contexts, logits of each prompt's last token)."""
    tables, ctx = [[] for _ in prompts], [0] * len(prompts)
    last = [None] * len(prompts)
    while any(c < len(p) for c, p in zip(ctx, prompts)):
        part = [p[c:c + chunk] for c, p in zip(ctx, prompts)]
        cu = starts(map(len, part))
        table = cache.grow(tables, [c + len(t) for c, t in zip(ctx, part)])
        logits = model.forward(torch.tensor(sum(part, []), device="cuda"), cache, table, ints(cu), ints(ctx), max_new=max(map(len, part)))
        for b, t in enumerate(part):
            if t:
                last[b] = logits[cu[b + 1] - 1]
        ctx = [c + len(t) for c, t in zip(ctx, part)]
    return tables, ctx, torch.stack(last)


def greedy(model, cache, prompts, steps):
    tables, ctx, logits = prefill(model, cache, prompts)
    out = [[] for _ in prompts]
    for step in range(steps):
        best = logits.argmax(-1)
        for o, t in zip(out, best.tolist()):
            o.append(t)
        if step + 1 < steps:
            table = cache.grow(tables, [c + 1 for c in ctx])
            logits = model.forward(best, cache, table, ints(list(range(len(prompts) + 1))), ints(ctx), max_new=1)
            ctx = [c + 1 for c in ctx]
    return out


def speculative(model, cache, prompts, steps, draft):
    """`draft(b, tokens so far)` proposes a tree: [(parent node, token)], parents first; node 0 is the last token that the
    model chose.  Returns the tokens, and the steps that they took."""
    tables, ctx, logits = prefill(model, cache, prompts)
    out = [[t] for t in logits.argmax(-1).tolist()]
    rounds = 0
    while min(map(len, out)) < steps:
        trees = [[(-1, o[-1])] + [(p, t) for p, t in draft(b, o)] for b, o in enumerate(out)]
        depth, seen = [], []
        for tree in trees:
            d, m = [], []
            for i, (p, _) in enumerate(tree):
                d.append(0 if p < 0 else d[p] + 1)
                m.append((0 if p < 0 else m[p]) | 1 << i)
            depth.append(d)
            seen.append(m)
        counts = [len(t) for t in trees]
        cu, words = starts(counts), -(-max(counts) // 32)
        signed = lambda w: w - (1 << 32) if w >> 31 else w  # noqa: E731
        mask = ints([[signed(m >> 32 * w & 0xFFFFFFFF) for w in range(words)] for ms in seen for m in ms])
        table = cache.grow(tables, [c + n for c, n in zip(ctx, counts)])
        positions = ints([c + x for c, d in zip(ctx, depth) for x in d])
        tokens = torch.tensor([t for tree in trees for _, t in tree], device="cuda")
        cu_t, ctx_t = ints(cu), ints(ctx)
        logits = model.forward(tokens, cache, table, cu_t, ctx_t, positions=positions, mask=mask, max_new=max(counts))
        choice = logits.argmax(-1).tolist()
        paths = []
        for b, tree in enumerate(trees):
            path = [0]
            while True:  # the child that the model itself would have chosen
                want = choice[cu[b] + path[-1]]
                child = [i for i, (p, t) in enumerate(tree) if p == path[-1] and t == want]
                out[b].append(want)
                if not child:
                    break
                path.append(child[0])
            paths.append(path)
        longest = max(map(len, paths))
        lens = paged.commit_path(cache.k, cache.v, table, cu_t, ctx_t, ints([p + [-1] * (longest - len(p)) for p in paths]))
        ctx = lens.tolist()
        rounds += 1
    return [o[:steps] for o in out], rounds


def beams(model, cache, prompt, steps, width):
    """The `width` best continuations of one prompt: (scores, token lists)."""
    tables, ctx, logits = prefill(model, cache, [prompt])
    # every hypothesis shares the prompt's full pages; the first step has one of them
    full = ctx[0] // cache.page_size
    open_pages = [cache.free.pop() for _ in range(width)]
    if len(tables[0]) > full:
        for p in open_pages:
            cache.k[:, p], cache.v[:, p] = cache.k[:, tables[0][full]], cache.v[:, tables[0][full]]
        cache.free += tables[0][full:]
    room = -(-(ctx[0] + steps) // cache.page_size) + 1
    table = ints([tables[0][:full] + [p] + [-1] * (room - full - 1) for p in open_pages])
    lens = ints([ctx[0]] * width)
    scores = torch.full((1, width), -float("inf"), device="cuda")
    scores[0, 0] = 0
    logits = logits[None].expand(1, width, -1).contiguous()
    one = ints(list(range(width + 1)))
    tokens = [[] for _ in range(width)]
    for step in range(steps):
        scores, parents, chosen = beam.select(logits, scores)
        tokens = [tokens[p] + [t] for p, t in zip(parents[0].tolist(), chosen[0].tolist())]
        if step + 1 == steps:
            break
        spare = [cache.free.pop() for _ in range(width)]
        before = pages_of(table)
        table, lens = beam.reorder(cache.k, cache.v, table, lens, parents, ints([spare]))
        # what no hypothesis holds any more is free again: the open pages of before, and full ones of dropped hypotheses
        cache.free += before - pages_of(table)
        logits = model.forward(chosen[0].long(), cache, table, one, lens, max_new=1).view(1, width, -1)
        lens = lens + 1
    return scores[0].tolist(), tokens


def main():
    model = Model()
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(model.vocab, (n,), generator=g).tolist() for n in (5, 37, 70)]
    plain = greedy(model, Cache(model, 64), prompts, 24)
    known = {b: plain[b] for b in range(len(prompts))}

    def draft(b, so_far):
        """Two branches: the continuation that greedy decoding found, with every third token spoiled, and noise."""
        ahead = known[b][len(so_far):len(so_far) + 5]
        chain = [(i, t if (len(so_far) + i) % 3 else (t + 1) % model.vocab) for i, t in enumerate(ahead)]
        return chain + [(0, 7), (len(chain) + 1, 9)]

    fast, rounds = speculative(model, Cache(model, 64), prompts, 24, draft)
    print(f"speculative: {rounds} steps for 24 tokens, the same as greedy decoding: {fast == plain}")
    scores, tokens = beams(model, Cache(model, 64), prompts[1], 12, 4)
    for s, t in zip(scores, tokens):
        print(f"beam {s:8.3f}  {t}")


if __name__ == "__main__":
    main()
