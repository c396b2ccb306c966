"""GPU tests of paged.evict: rows are chosen and copied, so everything is equal to the bit."""

import math
import random

import pytest
import torch

import paged_context_reference as C
import paged_reference as R
from test_gpu_paged import _bits, _ints

pytestmark = pytest.mark.gpu

F16, BF16, E4 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


def _check(seed, ctx, keep, recent=0, sinks=0, layers=2, kv=2, D=64, page=16, dtype=F16, rows=None, weights=None, spare=0, strided=False, wide=0,
           ties=0):
    import paged
    rng = random.Random(seed)
    g = torch.Generator().manual_seed(seed)
    B, pages_each = len(ctx), -(-keep // page)
    table, pages = R.make_pages(rng, ctx, page, B * (pages_each + spare))
    used = {p for row in table for p in row}
    free = [p for p in range(pages) if p not in used]
    fresh = [free[b * pages_each:(b + 1) * pages_each] + [0] * wide for b in range(B)]
    if strided:
        both = torch.randn(layers, pages, 2, kv, page, D, generator=g).to(dtype).cuda()
        k, v = both[:, :, 0], both[:, :, 1]
    else:
        k, v = (torch.randn(layers, pages, kv, page, D, generator=g).to(dtype).cuda() for _ in range(2))
    rows = max(ctx + [1]) + 2 if rows is None else rows
    w = torch.randn(layers, B, kv, rows, generator=g) if weights is None else weights(layers, B, kv, rows, g)
    if ties:
        w = (w * ties).round() / ties
    w = w.cuda()
    wk, wv = k.clone(), v.clone()
    want_w = torch.zeros(w.shape)
    for b, n in enumerate(ctx):
        for layer in range(layers):
            for h in range(kv):
                have = w[layer, b, h].tolist()
                stay = C.kept(have, n, keep, recent, sinks)
                for d, j in enumerate(stay):
                    if d < rows:
                        want_w[layer, b, h, d] = w[layer, b, h, j].cpu() if j < rows else 0.0
                if n > keep:
                    to, at = torch.tensor(range(keep)), torch.tensor(stay)
                    tp, sp = torch.tensor(fresh[b])[to // page], torch.tensor(table[b])[at // page]
                    for new, old in ((wk, k), (wv, v)):
                        new.view(torch.uint8 if dtype == E4 else dtype)[layer, tp.cuda(), h, (to % page).cuda()] = \
                            old.view(torch.uint8 if dtype == E4 else dtype)[layer, sp.cuda(), h, (at % page).cuda()]
    width = len(table[0])
    want_t = [row if n <= keep else (fresh[b][:pages_each] + [-1] * width)[:width] for b, (row, n) in enumerate(zip(table, ctx))]
    nt, nl, nw = paged.evict(k, v, _ints(table), _ints(ctx), w, _ints(fresh).reshape(B, -1), keep, recent=recent, sinks=sinks)
    assert nl.tolist() == [min(n, keep) for n in ctx] and nt.tolist() == want_t
    assert torch.equal(nw.cpu().nan_to_num(-77.0), want_w.nan_to_num(-77.0))
    assert torch.equal(_bits(k), _bits(wk)) and torch.equal(_bits(v), _bits(wv))


@pytest.mark.parametrize("dtype,D,page", [(F16, 128, 16), (BF16, 96, 32), (E4, 64, 1), (E4, 8, 16), (F16, 256, 64), (E4, 128, 128)])
def test_types_and_pages(cuda, dtype, D, page):
    _check(1, [100, 33, 0, 40, 7], 33, 8, 2, dtype=dtype, D=D, page=page)


@pytest.mark.parametrize("keep,recent,sinks", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (50, 25, 25), (50, 0, 0), (64, 64, 0), (64, 0, 64), (199, 3, 3)])
def test_counts(cuda, keep, recent, sinks):
    _check(2, [200, 64, 51], keep, recent, sinks)


@pytest.mark.parametrize("n", [1023, 1024, 1025, 2047, 2049, 8191, 8193, 20000, 33000])
def test_lengths(cuda, n):
    _check(3, [n, n // 2 + 1], n // 3 + 1, n // 10, 4, layers=1, kv=1, D=8, page=16)


@pytest.mark.parametrize("ties", [1, 2, 8])
def test_equal_weights_go_to_the_lower_row(cuda, ties):
    _check(4, [700, 1500, 90], 60, 10, 2, ties=ties)


def test_weights_of_every_kind(cuda):
    def odd(layers, B, kv, rows, g):
        w = torch.randn(layers, B, kv, rows, generator=g)
        pick = torch.randint(0, 9, w.shape, generator=g)
        for i, x in enumerate([math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-42, -1e-42, 3e38]):
            w[pick == i] = x
        return w
    for keep in (5, 40, 150, 290):
        _check(5, [300, 300], keep, 2, 1, weights=odd)
    _check(6, [300], 40, weights=lambda l, b, k, r, g: torch.zeros(l, b, k, r))
    _check(7, [300], 40, weights=lambda l, b, k, r, g: torch.full((l, b, k, r), math.nan))
    _check(8, [300], 40, weights=lambda l, b, k, r, g: torch.full((l, b, k, r), math.inf))


def test_rows_without_weights(cuda):
    """Rows past the weights' room count as the lowest."""
    _check(9, [100, 60], 30, 4, 1, rows=50)
    _check(10, [100, 60], 80, 4, 1, rows=50)
    _check(11, [100], 30, 4, 1, rows=0)


def test_strided_cache_and_wide_fresh(cuda):
    _check(12, [90, 30], 20, 5, strided=True, wide=3)


def test_many_sequences(cuda):
    rng = random.Random(13)
    _check(13, [rng.randrange(60) for _ in range(70)], 24, 4, 1, layers=1, kv=3, D=16)


def test_shared_pages_are_left_to_the_others(cuda):
    """Two sequences of the same pages: one may be cut, both are read as they were."""
    import paged
    k = torch.randn(1, 8, 1, 16, 64, device="cuda").half()
    v = torch.randn_like(k)
    table = _ints([[0, 1, 2], [0, 1, 3]])
    w = torch.rand(1, 2, 1, 48, device="cuda")
    old = k.clone()
    nt, nl, nw = paged.evict(k, v, table, _ints([48, 20]), w, _ints([[5, 6], [7, 4]]), 20)
    assert nt.tolist() == [[5, 6, -1], [0, 1, 3]] and nl.tolist() == [20, 20] and torch.equal(k[:, :5], old[:, :5]) and torch.equal(k[:, 7], old[:, 7])


def test_bad_pages(cuda):
    """Rows of missing pages are not copied, nor is anything to a missing page; contexts end with the table."""
    import paged
    k = torch.randn(1, 6, 1, 16, 64, device="cuda").half()
    v, before = torch.randn_like(k), k.clone()
    w = torch.arange(64, 0, -1, device="cuda").float().reshape(1, 1, 1, 64)
    nt, nl, nw = paged.evict(k, v, _ints([[0, 9, -1]]), _ints([10 ** 9]), w, _ints([[3, 77]]), 20)
    assert nt.tolist() == [[3, 77, -1]] and nl.tolist() == [20]
    assert torch.equal(k[0, 3, 0], before[0, 0, 0]) and torch.equal(k[0, [0, 1, 2, 4, 5]], before[0, [0, 1, 2, 4, 5]])
    assert torch.equal(nw[0, 0, 0, :20], w[0, 0, 0, :20]) and (nw[0, 0, 0, 20:] == 0).all()


def test_captured_and_other_streams(cuda):
    import paged
    g = torch.Generator(device="cuda").manual_seed(15)
    k, v = (torch.randn(2, 20, 2, 16, 64, generator=g, device="cuda").half() for _ in range(2))
    w = torch.rand(2, 1, 2, 160, generator=g, device="cuda")
    table, ctx, fresh = _ints([list(range(10))]), _ints([150]), _ints([[10, 11, 12]])
    want = [x.clone() for x in (*paged.evict(k, v, table, ctx, w, fresh, 40, 8, 2), k, v)]
    k[:, 10:], v[:, 10:] = 0, 0
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = paged.evict(k, v, table, ctx, w, fresh, 40, 8, 2, stream=s)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[:3]))
    # the fresh pages' first 40 rows: the others are not written
    assert torch.equal(k[:, 10:12], want[3][:, 10:12]) and torch.equal(k[:, 12, :, :8], want[3][:, 12, :, :8])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = paged.evict(k, v, table, ctx, w, fresh, 40, 8, 2)
    for n in (150, 30, 99):
        ctx.fill_(n)
        k[:, 10:] = 0
        graph.replay()
        torch.cuda.synchronize()
        first = [x.clone() for x in (*got, k)]
        k[:, 10:] = 0
        eager = paged.evict(k, v, table, ctx, w, fresh, 40, 8, 2)
        assert all(torch.equal(a, b) for a, b in zip(first, (*eager, k)))


def test_refusals(cuda):
    import paged
    k = torch.zeros(1, 4, 1, 16, 64, dtype=F16, device="cuda")
    w, table, ctx, fresh = torch.zeros(1, 1, 1, 32, device="cuda"), _ints([[0, 1]]), _ints([30]), _ints([[2]])
    paged.evict(k, k.clone(), table, ctx, w, fresh, 10)
    for kw in (dict(keep=0), dict(keep=17), dict(keep=10, recent=11), dict(keep=10, sinks=-1), dict(keep=2 ** 40), dict(keep=10, recent=5, sinks=6)):
        with pytest.raises(ValueError):
            paged.evict(k, k.clone(), table, ctx, w, fresh, **kw)
    for bad in (w.half(), w[0], w.cpu(), torch.zeros(1, 1, 2, 32, device="cuda"), torch.zeros(2, 1, 1, 32, device="cuda")):
        with pytest.raises(ValueError):
            paged.evict(k, k.clone(), table, ctx, bad, fresh, 10)
    with pytest.raises(ValueError):
        paged.evict(k, k.clone(), table, ctx, w, fresh.long(), 10)
