"""GPU tests of paged.weighted_attention with 17 to 64 rows (tokens x query heads) a kv head: drafted trees and a few tokens of a
chain behind contexts of several fully cached blocks and several ranges.  Limits as in test_gpu_paged_weighted.py and, for the
outputs, test_gpu_paged_attention.py."""

import pytest
import torch

from test_gpu_paged_attention import HALF, Case
from test_gpu_paged_weighted import _check as _check_sums

pytestmark = pytest.mark.gpu

F16, BF16, E4 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


def _case(seed, heads, kv, D, page, ctx, new, dtype, cache, mask):
    e4 = cache == E4
    return Case(seed, heads, kv, D, page, ctx, new, dtype, cache, mask, ks=0.0625 if e4 else 1.0, vs=0.3 if e4 else 1.0)


def _check(c):
    out, _ = _check_sums(c)
    want, spread = c.want()
    lim = HALF[c.dtype] * (want.abs() + spread) + 4e-5 * spread + 1e-7
    assert ((out.double().cpu() - want).abs() <= lim).all()


@pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, BF16), (F16, E4), (BF16, E4)])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("rows", [17, 32, 33, 48, 64])
def test_rows(cuda, rows, D, dtype, cache):
    """One query head a kv head, a tree; then the same rows as tokens of several heads, a chain where they divide."""
    _check(_case(rows + D, 2, 2, D, 16, [100, 1300], [rows, rows - 1], dtype, cache, "tree"))
    group = next((g for g in (4, 3, 2) if rows % g == 0), 1)
    _check(_case(rows + D + 1, 2 * group, 2, D, 32, [640, 0, 257], [rows // group, 1, 2], dtype, cache, None))


@pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, E4)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_long_contexts(cuda, D, dtype, cache):
    _check(_case(D, 8, 1, D, 64, [2000, 4096], [3, 4], dtype, cache, "tree"))
    _check(_case(D + 1, 8, 1, D, 16, [4095], [8], dtype, cache, None))


def test_many_sequences(cuda):
    _check(_case(5, 8, 2, 128, 16, [(37 * i) % 300 for i in range(70)], [1 + (5 * i) % 8 for i in range(70)], F16, F16, "tree"))


def test_the_same_sums_every_time(cuda):
    import paged
    from test_gpu_paged_attention import _ints, _words
    c = _case(6, 16, 2, 128, 16, [1500, 900, 64, 3], [5, 8, 8, 2], F16, F16, "tree")
    args = (c.q, c.k, c.v, _ints(c.table).reshape(4, -1), _ints(c.cu), _ints(c.ctx))
    first = None
    for _ in range(50):
        out, sums = paged.weighted_attention(*args, torch.zeros(4, 2, 1520, device="cuda"), mask=_words(c.masks, 1), max_new=8)
        first = first or (out.clone(), sums.clone())
        assert torch.equal(out, first[0]) and torch.equal(sums, first[1])
