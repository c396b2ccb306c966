"""GPU tests of paged.evict on sequences that miss pages of their tables (a window's dropped pages, -1): rows without a page are not
kept and not seen afterwards.  Rows are chosen and copied, so everything is equal to the bit; the attention over the result
is held to test_gpu_paged_attention.py's limit."""

import math
import random

import pytest
import torch

from test_gpu_paged import _bits, _ints

pytestmark = pytest.mark.gpu

F16, BF16, E4 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


def kept(weights, n, keep, recent, sinks, has):
    """The rows that stay, ascending; has(j): row j has a page."""
    if n <= keep:
        return list(range(n))

    def key(j):
        w = weights[j] if j < len(weights) else -math.inf
        return -math.inf if math.isnan(w) else w

    ends = [j for j in [*range(sinks), *range(n - recent, n)] if has(j)]
    between = sorted((j for j in range(sinks, n - recent) if has(j)), key=lambda j: (-key(j), j))
    return sorted(ends + between[:keep - len(ends)])


def _check(seed, ctx, gaps, keep, recent=0, sinks=0, layers=2, kv=2, D=64, page=16, dtype=F16, rows=None, ties=0, few=False):
    """gaps: the places of each sequence's missing pages in its table; few: a sequence may have fewer rows than `keep`."""
    import paged
    rng = random.Random(seed)
    g = torch.Generator().manual_seed(seed)
    B, each, width = len(ctx), -(-keep // page), max(-(-n // page) for n in ctx)
    ids = list(range(B * (width + each) + 1))
    rng.shuffle(ids)
    table = [[ids.pop() if p < -(-n // page) else -1 for p in range(width)] for n in ctx]
    for row, missing in zip(table, gaps):
        for p in missing:
            row[p] = rng.choice([-1, 10 ** 6])
    fresh = [[ids.pop() for _ in range(each)] for _ in range(B)]
    pages = B * (width + each) + 1
    k, v = (torch.randn(layers, pages, kv, page, D, generator=g).to(dtype).cuda() for _ in range(2))
    for x in (k, v):  # what the fresh pages held before
        x.view(torch.uint8 if dtype == E4 else dtype)[:, [p for f in fresh for p in f]] = 0x7F if dtype == E4 else float("nan")
    rows = max(ctx) + 2 if rows is None else rows
    w = torch.randn(layers, B, kv, rows, generator=g)
    if ties:
        w = (w * ties).round() / ties
    w = w.cuda()
    wk, wv, want_w, stays = k.clone(), v.clone(), torch.zeros(w.shape), {}
    for b, n in enumerate(ctx):
        for layer in range(layers):
            for h in range(kv):
                have = w[layer, b, h].tolist()
                stay = stays[layer, b, h] = kept(have, n, keep, recent, sinks, lambda j: 0 <= table[b][j // page] < pages)
                for d, j in enumerate(stay):
                    if d < rows:
                        want_w[layer, b, h, d] = have[j] if j < rows else 0.0
                if n > keep and stay:
                    to, at = torch.tensor(range(len(stay))), torch.tensor(stay)
                    tp, sp = torch.tensor(fresh[b])[to // page], torch.tensor(table[b])[at // page]
                    for new, old in ((wk, k), (wv, v)):
                        new.view(torch.uint8 if dtype == E4 else dtype)[layer, tp.cuda(), h, (to % page).cuda()] = \
                            old.view(torch.uint8 if dtype == E4 else dtype)[layer, sp.cuda(), h, (at % page).cuda()]
    lens = [len(stays[0, b, 0]) for b in range(B)]
    assert few or all(x == min(n, keep) for x, n in zip(lens, ctx))
    want_t = [row if n <= keep else (fresh[b][:-(-lens[b] // page)] + [-1] * width)[:width] for b, (row, n) in enumerate(zip(table, ctx))]
    nt, nl, nw = paged.evict(k, v, _ints(table), _ints(ctx), w, _ints(fresh), keep, recent=recent, sinks=sinks)
    assert nl.tolist() == lens and nt.tolist() == want_t
    assert torch.equal(nw.cpu(), want_w)
    assert torch.equal(_bits(k), _bits(wk)) and torch.equal(_bits(v), _bits(wv))
    return k, v, nt, nl, stays, table


@pytest.mark.parametrize("dtype,D,page", [(F16, 128, 16), (BF16, 96, 32), (E4, 64, 16), (E4, 8, 16)])
def test_types_and_pages(cuda, dtype, D, page):
    _check(1, [7 * page, 5 * page + 3, 4 * page, 9], [[1, 3], [], [0], []], 2 * page + 1, 8, 2, dtype=dtype, D=D, page=page)


@pytest.mark.parametrize("keep,recent,sinks", [(1, 0, 0), (1, 1, 0), (20, 0, 20), (20, 20, 0), (40, 25, 15), (40, 0, 0), (63, 40, 20)])
def test_rows_that_would_always_stay(cuda, keep, recent, sinks):
    """The first and the last rows too, and others take their places."""
    _check(2, [200, 164, 130, 140], [[0, 12], [1, 9], [0, 2, 8], [8]], keep, recent, sinks, few=True)


@pytest.mark.parametrize("keep", [31, 32, 33, 40, 64])
def test_shorter_than_keep(cuda, keep):
    """A sequence with fewer rows than `keep`, or none, ends with them."""
    _check(3, [100, 100, 65], [[1, 2, 4, 6], [0, 1, 2, 3, 4, 5, 6], [0, 1, 2, 3]], keep, 8, 4, few=True)


@pytest.mark.parametrize("n", [4097, 9000, 20000, 33000])
def test_lengths(cuda, n):
    """Every variant by the table's width."""
    rng = random.Random(n)
    pages = -(-n // 64)
    _check(4, [n, n - 70], [rng.sample(range(pages), pages // 4), []], n // 4, n // 20, 4, layers=1, kv=2, D=8, page=64, rows=n - 5)


@pytest.mark.parametrize("ties", [1, 2])
def test_equal_weights_go_to_the_lower_row(cuda, ties):
    _check(5, [700, 900], [[3, 7, 8, 30], [0]], 200, 10, 2, ties=ties)


def test_weights_shorter_than_the_rows(cuda):
    _check(6, [100, 90], [[2], [4]], 60, 4, 1, rows=50)


@pytest.mark.parametrize("keep", [40, 60])
def test_attention_afterwards(cuda, keep):
    """Sees the kept rows and nothing else."""
    import paged
    n, kv, heads, D, page = 112, 2, 4, 64, 16
    k, v, nt, nl, stays, table = _check(7, [n], [[0, 2, 4, 5]], keep, 8, 4, layers=1, kv=kv, D=D, page=page, few=True)
    q = torch.randn(1, heads, D, generator=torch.Generator().manual_seed(8)).half().cuda()
    out = paged.tree_attention(q, k[0], v[0], nt, _ints([0, 1]), nl, mask=_ints([[0]]), max_new=1)
    for h in range(heads):
        at = torch.tensor(stays[0, 0, h // 2])
        pages = torch.tensor(table[0])[at // page].cuda()
        kh, vh = (x[0, pages, h // 2, (at % page).cuda()].double().cpu() for x in (k, v))
        p = torch.softmax(kh @ q[0, h].double().cpu() / math.sqrt(D), 0)
        want, spread = p @ vh, p @ vh.abs()
        assert ((out[0, h].double().cpu() - want).abs() <= 2.0 ** -11 * (want.abs() + spread) + 4e-5 * spread + 1e-7).all()
