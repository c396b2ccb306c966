"""GPU tests of paged.tree_attention where the keys are cut into ranges, beyond what few rows and short contexts reach: tiles of
128 rows over several ranges, missing pages and infinite values in later ones, other head sizes and small pages over several.
Tolerances and restatement as in test_gpu_paged_attention.py."""

import pytest
import torch

from test_gpu_paged_attention import BF16, E4, F16, Case

pytestmark = pytest.mark.gpu

TYPES = [(F16, F16), (BF16, BF16), (F16, E4), (BF16, E4)]


def _tiled(c, kv, least=2):
    """The call takes 128-row tiles, and a sequence at least `least` ranges.  A range is four steps of 64 keys where the whole call
    has no more than four steps for each of 256 workgroups, and no more ranges than those: any occupancy allows it."""
    group = c.heads // kv
    assert max(c.new) * group > (64 if c.q.shape[2] <= 128 else 16)
    steps = [-(-(x + n) // 64) if n else 0 for x, n in zip(c.ctx, c.new)]
    tiles = [-(-n * group // 128) for n in c.new]
    assert sum(s * t for s, t in zip(steps, tiles)) * kv <= 4 * 256
    assert sum(-(-s // 4) * t for s, t in zip(steps, tiles)) * kv <= 256
    assert max(-(-s // 4) for s in steps) >= least
    return c


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_chains_over_ranges(cuda, D, dtype, cache):
    _tiled(Case(D + 3, 8, 2, D, 64, [900, 0, 5], [40, 70, 0], dtype, cache, None, ks=0.0625 if cache == E4 else 1.0), 2, 4).check()


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_trees_over_ranges(cuda, D, dtype, cache):
    _tiled(Case(D + 4, 8, 2, D, 16, [700, 300, 1500], [33, 17, 5], dtype, cache, "tree", vs=0.3 if cache == E4 else 1.0), 2, 6).check()


def test_long_chain_past_its_first_rows_ranges(cuda):
    """Ranges that hold keys of later rows alone: the first row tiles see none of them."""
    _tiled(Case(50, 4, 1, 64, 32, [0], [600], mask=None), 1, 3).check()


@pytest.mark.parametrize("D,dtype,cache", [(64, F16, F16), (128, BF16, BF16), (128, F16, E4), (256, F16, F16)])
@pytest.mark.parametrize("page", [16, 64])
def test_missing_pages_of_later_tiles(cuda, D, dtype, cache, page):
    c = _tiled(Case(51, 8, 2, D, page, [1200, 640], [40, 18], dtype, cache, "tree"), 2, 5)
    for row, gone in ((0, (3, 1040 // page, 1215 // page)), (1, (0, 500 // page))):
        for p in gone:
            c.table[row][p] = -1 if p % 2 else c.pages + p
    c.check()


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16), (256, F16)])
def test_missing_pages_at_either_end(cuda, D, dtype):
    c = _tiled(Case(52, 8, 2, D, 32, [1000], [40], dtype, None, None), 2, 4)
    c.table[0][0] = -1
    c.table[0][-1] = -1
    c.check()


@pytest.mark.parametrize("D,dtype,cache", [(64, F16, F16), (128, BF16, BF16), (96, F16, F16), (256, BF16, BF16)])
def test_infinite_value_in_a_later_range(cuda, D, dtype, cache):
    c = _tiled(Case(53, 8, 2, D, 16, [1000], [40], dtype, cache, "tree"), 2, 4)
    clean = c.run().float()
    c.v[c.table[0][900 // 16], :, 900 % 16, 7] = float("inf")
    got = c.run().float()
    keep = [d for d in range(D) if d != 7]
    assert (got[:, :, 7] == float("inf")).all()
    # rows that were taken another way: the same values up to a rounding of the weights and one of the output
    lim = 2.0 ** (-9 if dtype == F16 else -6)
    assert ((got - clean)[:, :, keep].abs() <= lim * (1 + clean[:, :, keep].abs())).all()


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, F16), (96, BF16), (256, F16)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_unseen_values_in_the_last_range(cuda, D, dtype, value):
    """A new row's NaN or infinite key and value reach those alone that see it."""
    n = 40
    c = _tiled(Case(54, 8, 2, D, 16, [1000], [n], dtype, None, "tree"), 2, 4)
    clean = c.run().float()
    bad = 30
    pg, slot = c.table[0][(1000 + bad) // 16], (1000 + bad) % 16
    lim = 2.0 ** (-9 if dtype == F16 else -6)
    for cache in (c.k, c.v):
        keep = cache[pg, :, slot].clone()
        cache[pg, :, slot] = value
        got = c.run().float()
        cache[pg, :, slot] = keep
        unseen = [t for t in range(n) if not (c.masks[t] >> bad) & 1]
        assert unseen and ((got - clean)[unseen].abs() <= lim * (1 + clean[unseen].abs())).all()
    c.v[pg, :, slot] = value
    got = c.run().float()
    seen = [t for t in range(n) if (c.masks[t] >> bad) & 1]
    assert seen and (got[seen].isnan() if value != value else got[seen] == value).all()


@pytest.mark.parametrize("D", [8, 40, 80, 160, 200, 248])
def test_other_head_sizes_over_ranges(cuda, D):
    """Heads whose quarter does not divide a workgroup: the ranges (64 keys each) are joined by uneven groups of threads."""
    Case(55, 6, 2, D, 16, [300, 70, 0], [3, 9, 1], mask="tree").check()
    Case(56, 6, 2, D, 16, [700], [2], BF16, E4, mask=None).check()


@pytest.mark.parametrize("page", [1, 8])
def test_small_pages_over_ranges(cuda, page):
    Case(57, 4, 1, 128, page, [500, 3], [5, 2], mask="tree").check()


def test_many_single_tokens_without_a_bound(cuda):
    """Without max_new the tokens of all sequences bound those of one: 128-row tiles with a few rows each."""
    c = Case(62, 8, 1, 64, 16, [(37 * i) % 400 for i in range(40)], [1] * 40, mask=None)
    c.check(max_new=None)
    c.check()


def test_repeats_are_equal_to_the_bit(cuda):
    """Partial results are joined in a fixed order, whichever workgroup comes first."""
    for c in (_tiled(Case(59, 8, 2, 128, 32, [1500, 20], [40, 70], mask="tree"), 2, 4), Case(60, 8, 2, 128, 16, [4000, 9], [13, 2], cache=E4, mask="tree"),
              Case(61, 6, 2, 80, 16, [700], [5], mask="tree")):
        first = c.run().clone()
        for _ in range(5):
            assert torch.equal(c.run(), first)
