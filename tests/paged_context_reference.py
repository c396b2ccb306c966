"""Plain 64-bit restatement, on the CPU, of the paged cache's normed append, weight sums and eviction (test infrastructure);
`paged_reference` has what they build on."""

import math

import torch


def normed(x, weight, eps):
    """x [heads, D] float64, each head normed; weight None: as it is."""
    return x if weight is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight


def rotate_axes(x, pos, base, rotary, neox, axes):
    """x [heads, D] float64; pos: one position per axis."""
    x = x.clone()
    half = rotary // 2
    for i in range(half):
        a = pos[axes[i]] * base ** (-2.0 * i / rotary)
        c, s = math.cos(a), math.sin(a)
        i0, i1 = (i, i + half) if neox else (2 * i, 2 * i + 1)
        f, g = x[:, i0].clone(), x[:, i1].clone()
        x[:, i0], x[:, i1] = f * c - g * s, f * s + g * c
    return x


def sums(q, k_cache, table, cu, ctx, page, mask=None, scale=None, most=None):
    """{(sequence, row): [kv_heads] float64}: what every row of a sequence gets from its new tokens."""
    T, heads, D = q.shape
    kv = k_cache.shape[1]
    group = heads // kv
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    got = {}
    for b in range(len(ctx)):
        n = cu[b + 1] - cu[b]
        rows = ctx[b] + n
        have = [i for i in range(min(rows, len(table[b]) * page)) if 0 <= table[b][i // page] < k_cache.shape[0]]
        total = torch.zeros(rows, kv, dtype=torch.float64)
        k = torch.stack([k_cache[table[b][i // page], :, i % page] for i in have]) if have else None
        for i in range(n if most is None else min(n, most)):
            t = cu[b] + i
            seen = [x for x, j in enumerate(have) if j < ctx[b] or ((mask[t] >> (j - ctx[b])) & 1 if mask is not None else j - ctx[b] <= i)]
            if not seen:
                continue
            s = (k[seen].repeat_interleave(group, 1) * q[t]).sum(-1) * scale
            total[[have[x] for x in seen]] += torch.softmax(s, 0).reshape(len(seen), kv, group).sum(-1)
        for j in range(rows):
            got[b, j] = total[j]
    return got


def kept(weights, n, keep, recent, sinks):
    """The rows that stay of n, ascending; weights: a list of floats (rows past its end count as -inf)."""
    if n <= keep:
        return list(range(n))

    def key(j):
        w = weights[j] if j < len(weights) else -math.inf
        return -math.inf if math.isnan(w) else w

    middle = sorted(range(sinks, n - recent), key=lambda j: (-key(j), j))[:keep - sinks - recent]
    return sorted(list(range(sinks)) + middle + list(range(n - recent, n)))
