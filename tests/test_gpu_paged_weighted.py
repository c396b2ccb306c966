"""GPU tests of paged.weighted_attention against the 64-bit restatements in paged_reference.py (outputs) and
paged_context_reference.py (sums).

Tolerance of a sum: a weight is off by 4e-5 of itself for fp32 scores up to about 30 (test_gpu_paged_attention.py; the sum that it
is divided by is within that), sums of up to 2^12 fp32 terms by 2^-24 of the running sum a term at most, in practice far
less: 2^-16 of the sum; adding the old sum rounds once more."""

import random

import pytest
import torch

import paged_context_reference as C
from test_gpu_paged_attention import Case, _ints

pytestmark = pytest.mark.gpu

F16, BF16, E4 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


def _check(c, rows=None, in_place=False, scale=None, max_new=None, strided=False):
    import paged
    words = max(1, -(-max(c.new) // 32))
    from test_gpu_paged_attention import _words
    kv = c.k.shape[1]
    rows = max(x + n for x, n in zip(c.ctx, c.new)) + 3 if rows is None else rows
    g = torch.Generator().manual_seed(1)
    old = torch.rand(len(c.ctx), kv, rows, generator=g).cuda()
    for b, x in enumerate(c.ctx):  # whatever is behind the cached rows is not read
        old[b, :, x:] = float("nan")
    if strided:
        wide = torch.full((len(c.ctx), 2, kv, rows + 5), 3.0, device="cuda")
        wide[:, 1, :, 2:2 + rows] = old
        old = wide[:, 1, :, 2:2 + rows]
    start = old.clone()
    new = old if in_place else torch.full_like(start, 5.0)
    out, got = paged.weighted_attention(c.q, c.k, c.v, _ints(c.table).reshape(len(c.ctx), -1), _ints(c.cu), _ints(c.ctx), old,
                                        weights_out=None if in_place else new, mask=None if c.masks is None else _words(c.masks, words),
                                        max_new=max(c.new) if max_new is None else max_new, scale=scale, k_scale=c.ks, v_scale=c.vs)
    assert got.data_ptr() == new.data_ptr()
    want = C.sums(c.q.double().cpu(), c.k.float().double().cpu() * c.ks, c.table, c.cu, c.ctx, c.page, c.masks, scale, max_new)
    have, before = got.double().cpu(), start.double().cpu()
    for b, x in enumerate(c.ctx):
        held = x + c.new[b]
        for j in range(rows):
            if j >= held:  # as it was
                assert torch.equal(have[b, :, j].nan_to_num(-1.0), before[b, :, j].nan_to_num(-1.0) if in_place else torch.full((kv,), 5.0).double())
                continue
            s = want[b, j]
            base = before[b, :, j] if j < x else torch.zeros(kv, dtype=torch.float64)
            lim = 4e-5 * s + 2.0 ** -16 * s + 2.0 ** -23 * (base + s) + 1e-9
            assert ((have[b, :, j] - base - s).abs() <= lim).all(), (b, j, have[b, :, j], base + s)
    if strided:
        assert (wide[:, 0] == 3).all() and (wide[:, 1, :, :2] == 3).all() and (wide[:, 1, :, 2 + rows:] == 3).all()
    return out, got


def _both(c, **kw):
    out, got = _check(c, **kw)
    if kw.get("max_new") is None:
        assert torch.equal(out, c.run(**({"scale": kw["scale"]} if kw.get("scale") else {})))
    return out, got


@pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, BF16), (F16, E4), (BF16, E4)])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_decode_step(cuda, D, dtype, cache):
    e4 = cache == E4
    _both(Case(D, 8, 2, D, 16, [0, 1, 63, 200], [1, 1, 1, 1], dtype, cache, None, ks=0.0625 if e4 else 1.0, vs=0.3 if e4 else 1.0))


@pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, BF16), (F16, E4), (BF16, E4)])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_trees(cuda, D, dtype, cache):
    _both(Case(D + 1, 8, 2, D, 32, [0, 70, 130], [13, 40, 1], dtype, cache, "tree", ks=0.0625 if cache == E4 else 1.0))


@pytest.mark.parametrize("heads,kv", [(32, 32), (32, 8), (16, 2), (12, 4), (8, 1), (5, 1), (34, 2), (3, 3), (64, 1)])
@pytest.mark.parametrize("n", [1, 3, 21])
def test_head_groups(cuda, heads, kv, n):
    _both(Case(heads + n, heads, kv, 64, 16, [50, 7], [n, max(1, n - 2)], mask="tree"))


@pytest.mark.parametrize("page", [1, 2, 8, 16, 64, 256])
def test_page_sizes(cuda, page):
    _both(Case(page, 4, 1, 128, page, [0, 127, 130, 64], [33, 2, 1, 5], mask="tree"))


@pytest.mark.parametrize("D", [8, 40, 112, 248])
def test_other_head_sizes(cuda, D):
    _both(Case(D, 6, 2, D, 16, [33, 0], [4, 9], mask="tree"))
    _both(Case(D, 6, 2, D, 16, [33, 0], [4, 9], BF16, E4, mask=None))


@pytest.mark.parametrize("n", [2, 31, 33, 64, 65, 128, 150])
def test_masks_that_leave_rows_empty(cuda, n):
    _both(Case(n, 4, 2, 64, 16, [3, 0], [n, (n + 1) // 2], mask="random"))


@pytest.mark.parametrize("D", [64, 128, 256])
def test_chunks_of_prompts(cuda, D):
    _both(Case(4, 8, 2, D, 16, [100, 0, 31], [150, 300, 5], BF16, mask=None))


def test_long_contexts(cuda):
    """Several ranges a sequence."""
    _both(Case(5, 8, 1, 128, 16, [6000, 40, 3000], [1, 1, 2], mask=None))
    _both(Case(6, 4, 1, 64, 32, [5000], [40], mask="tree"))


def test_in_place_strided_and_short_sums(cuda):
    _both(Case(7, 8, 2, 64, 16, [20, 90], [3, 5], mask="tree"), in_place=True)
    _both(Case(8, 8, 2, 64, 16, [20, 90], [3, 5], mask="tree"), in_place=True, strided=True)
    _both(Case(9, 8, 2, 128, 16, [20, 90], [3, 5], mask=None), rows=37)
    _both(Case(9, 8, 2, 128, 16, [20, 90], [3, 5], mask=None), rows=1)


def test_sequences_without_new_tokens(cuda):
    """Their sums are passed on."""
    _both(Case(10, 8, 2, 64, 16, [20, 0, 40], [0, 0, 3], mask=None))


def test_tokens_past_max_new(cuda):
    _check(Case(11, 8, 2, 64, 16, [20, 5], [2, 9], mask=None), max_new=4)


def test_scales(cuda):
    _both(Case(12, 8, 2, 128, 16, [300], [2], q_scale=4.0, mask=None), scale=0.3)
    _both(Case(13, 8, 2, 64, 16, [300], [40], mask="tree"), scale=-0.2)


def test_nan_and_missing_pages(cuda):
    """Rows that nobody sees may hold NaN; rows without a page get nothing, and keep what they had."""
    c = Case(14, 8, 2, 64, 16, [70, 40], [2, 3], mask="tree")
    c.table[0][2] = -1
    c.table[1][1] = 10 ** 6
    _both(c)
    c = Case(15, 8, 2, 64, 16, [30], [3], mask="tree")
    c.masks = [1, 2, 1 | 4]
    row = c.ctx[0] + 1
    c.k[c.table[0][row // 16], :, row % 16] = float("nan")
    import paged
    sums = torch.zeros(1, 2, 40, device="cuda")
    from test_gpu_paged_attention import _words
    paged.weighted_attention(c.q, c.k, c.v, _ints(c.table), _ints(c.cu), _ints(c.ctx), sums, mask=_words(c.masks, 1), max_new=3)
    assert sums[0, :, row].isnan().all() and not sums[0, :, [j for j in range(40) if j != row]].isnan().any() or \
        sums[0, :, :30].isnan().all()  # the token that sees the row itself: its weights are NaN wherever it looks


def test_repeats_captured_and_other_streams(cuda):
    import paged
    c = Case(16, 16, 2, 128, 16, [900, 40, 333], [1, 1, 1], mask=None)
    args = (c.q, c.k, c.v, _ints(c.table), _ints(c.cu), _ints(c.ctx))
    zero = lambda: torch.zeros(3, 2, 960, device="cuda")  # noqa: E731
    out, sums = paged.weighted_attention(*args, zero(), max_new=1)
    s = torch.cuda.Stream()
    w = zero()
    s.wait_stream(torch.cuda.current_stream())
    o2, w2 = paged.weighted_attention(*args, w, max_new=1, stream=s)
    s.synchronize()
    assert torch.equal(out, o2) and torch.equal(sums, w2)
    old, new, o3 = zero(), zero(), torch.empty_like(out)
    paged.weighted_attention(*args, old, weights_out=new, max_new=1, out=o3)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        paged.weighted_attention(*args, old, weights_out=new, max_new=1, out=o3)
    for ctx in ([900, 40, 333], [17, 0, 332], [500, 39, 1]):
        args[5].copy_(_ints(ctx))
        new.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = o3.clone(), new.clone()
        want = paged.weighted_attention(*args, zero(), max_new=1)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals(cuda):
    import paged
    c = Case(17, 4, 2, 64, 16, [10], [1], mask=None)
    args = (c.q, c.k, c.v, _ints(c.table), _ints(c.cu), _ints(c.ctx))
    w = torch.zeros(1, 2, 16, device="cuda")
    for bad in (w.half(), w[:, :1], w[0], w.cpu(), torch.zeros(1, 2, 32, device="cuda")[..., ::2]):
        with pytest.raises(ValueError, match="weights"):
            paged.weighted_attention(*args, bad)
    with pytest.raises(ValueError, match="weights_out"):
        paged.weighted_attention(*args, w, weights_out=torch.zeros(1, 2, 17, device="cuda"))
