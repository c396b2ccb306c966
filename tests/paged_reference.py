"""Plain 64-bit restatement of the paged-cache and beam operators on the CPU, row by row (test infrastructure).

Index tensors are lists of Python ints; caches are float64 tensors [pages, kv_heads, page_size, head_dim]."""

import math

import torch


def make_pages(rng, lens, page, extra_pages=0):
    """(table as lists padded with -1, page count): pages in random order."""
    need = [-(-n // page) for n in lens]
    ids = list(range(sum(need) + extra_pages))
    rng.shuffle(ids)
    width = max(need + [1])
    table, at = [], 0
    for k in need:
        table.append(ids[at:at + k] + [-1] * (width - k))
        at += k
    return table, sum(need) + extra_pages


def rotate(x, pos, base, rotary, neox):
    """x [heads, D] float64 at one position."""
    x = x.clone()
    half = rotary // 2
    for i in range(half):
        a = pos * base ** (-2.0 * i / rotary)
        c, s = math.cos(a), math.sin(a)
        i0, i1 = (i, i + half) if neox else (2 * i, 2 * i + 1)
        f, g = x[:, i0].clone(), x[:, i1].clone()
        x[:, i0], x[:, i1] = f * c - g * s, f * s + g * c
    return x


def rows(cache, table_row, page, n):
    return torch.stack([cache[table_row[i // page], :, i % page] for i in range(n)]) if n else cache.new_zeros((0, cache.shape[1], cache.shape[3]))


def attention(q, k_cache, v_cache, table, cu, ctx, page, mask=None, scale=None):
    """(out, spread) [T, heads, D] float64: spread = sum p |v| / sum p, what a relative error of the weights acts on.
    mask: list of Python ints per token (bit j: new token j is seen)."""
    T, heads, D = q.shape
    kv = k_cache.shape[1]
    group = heads // kv
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out, spread = torch.zeros(T, heads, D, dtype=torch.float64), torch.zeros(T, heads, D, dtype=torch.float64)
    for b in range(len(ctx)):
        n = cu[b + 1] - cu[b]
        if n == 0:
            continue
        total = min(ctx[b] + n, len(table[b]) * page)
        valid = [i for i in range(total) if 0 <= table[b][i // page] < k_cache.shape[0]]
        k = torch.stack([k_cache[table[b][i // page], :, i % page] for i in valid]) if valid else None
        v = torch.stack([v_cache[table[b][i // page], :, i % page] for i in valid]) if valid else None
        for i in range(n):
            t = cu[b] + i
            seen = [x for x, j in enumerate(valid) if j < ctx[b] or ((mask[t] >> (j - ctx[b])) & 1 if mask is not None else j - ctx[b] <= i)]
            if not seen:
                continue
            ks, vs = k[seen].repeat_interleave(group, 1), v[seen].repeat_interleave(group, 1)
            s = (ks * q[t]).sum(-1) * scale  # [keys, heads]
            p = torch.softmax(s, 0)
            out[t] = (p[..., None] * vs).sum(0)
            spread[t] = (p[..., None] * vs.abs()).sum(0)
    return out, spread


def select(logits, scores):
    """(scores, parents, tokens) of logits [B, W, V] and scores [B, W], float64 in, lists out."""
    B, W, V = logits.shape
    res = []
    for b in range(B):
        lse = torch.logsumexp(logits[b], -1, keepdim=True)
        total = (scores[b][:, None] + (logits[b] - lse)).reshape(-1)
        total = torch.where(total.isnan(), torch.full_like(total, -math.inf), total)
        order = torch.sort(total, descending=True, stable=True)
        res.append((order.values[:W], order.indices[:W] // V, order.indices[:W] % V))
    return tuple(torch.stack([r[i] for r in res]) for i in range(3))
