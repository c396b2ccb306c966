"""GPU tests of what a token with a NaN score does to the sums of paged.weighted_attention: the rows that it sees get NaN, every
other row what the other tokens give it, whichever kernel forms the sums.  Limits as in test_gpu_paged_weighted.py."""

import pytest
import torch

import paged_context_reference as C
from test_gpu_paged_attention import Case, _ints, _words

pytestmark = pytest.mark.gpu

F16, BF16, E4 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


@pytest.mark.parametrize("what", ["key", "query"])
@pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, E4)])
# stored scores, keys again with one and more row tiles, tiles of keys, the vector ALUs
@pytest.mark.parametrize("heads,D", [(4, 128), (4, 256), (8, 64), (24, 128), (40, 64), (64, 128), (8, 40)])
def test_only_what_the_token_sees(cuda, heads, D, dtype, cache, what):
    import paged
    c = Case(heads + D, heads, 2, D, 16, [70, 33], [3, 3], dtype, cache, mask="tree")
    c.masks = [1, 2, 1 | 4] * 2
    c.table[0][2] = -1  # rows 32 .. 47
    if what == "key":
        c.k.view(torch.uint8 if cache == E4 else c.k.dtype)[c.table[0][71 // 16], :, 71 % 16] = 0x7F if cache == E4 else float("nan")
    else:
        c.q[1, :, 5] = float("nan")
    old = torch.rand(2, 2, 80, generator=torch.Generator().manual_seed(1)).cuda()
    new = torch.full_like(old, 5.0)
    paged.weighted_attention(c.q, c.k, c.v, _ints(c.table), _ints(c.cu), _ints(c.ctx), old, weights_out=new, mask=_words(c.masks, 1), max_new=3)
    want = C.sums(c.q.double().cpu(), c.k.float().double().cpu(), c.table, c.cu, c.ctx, c.page, c.masks)
    got, before = new.double().cpu(), old.double().cpu()
    for b, x in enumerate(c.ctx):
        for j in range(80):
            if j >= x + 3:
                assert (got[b, :, j] == 5).all()
                continue
            s, base = want[b, j], before[b, :, j] if j < x else torch.zeros(2, dtype=torch.float64)
            nan = b == 0 and (j < 70 and j // 16 != 2 or j == 71)
            assert s.isnan().all() == nan and got[b, :, j].isnan().all() == nan, (b, j, got[b, :, j], s)
            if not nan:
                assert ((got[b, :, j] - base - s).abs() <= 6e-5 * s + 2.0 ** -23 * (base + s) + 1e-9).all(), (b, j, got[b, :, j], base + s)
