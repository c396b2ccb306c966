"""GPU tests of paged.shared_attention: its definition is tree_attention's over the sequences' own tables, so it is held against the
64-bit restatement in paged_reference.py.  The tolerance of an output is that of tree_attention (test_gpu_paged_attention.py): its own
rounding, the weights' rounding before the second product, 4e-5 of sum p |v|; joining two more partial results in fp32 is
within the last."""

import random

import pytest
import torch

import paged_reference as R
from test_gpu_paged_attention import HALF, _ints, _tree_mask, _words

pytestmark = pytest.mark.gpu

F16, BF16, E4 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


class Case:
    """Groups of `sizes` sequences behind `prefix` rows each, then rows of their own."""

    def __init__(self, seed, heads, kv, D, page, sizes, prefix, own, new, dtype=F16, cache=None, mask=None, ks=1.0, vs=1.0, q_scale=1.0):
        rng = random.Random(seed)
        g = torch.Generator().manual_seed(seed)
        cache = cache or dtype
        self.page, self.dtype, self.heads, self.new, self.ks, self.vs = page, dtype, heads, new, ks, vs
        group = [i for i, n in enumerate(sizes) for _ in range(n)]
        self.ctx = [prefix[i] + o for i, o in zip(group, own)]
        self.cu, self.first = [0], [0]
        for n in new:
            self.cu.append(self.cu[-1] + n)
        for n in sizes:
            self.first.append(self.first[-1] + n)
        self.shared = [p // page * page for p in prefix]
        # a sequence's own pages, and its group's ahead of them
        lead, pages = R.make_pages(rng, self.shared, page)
        own_table, count = R.make_pages(rng, [c + n - self.shared[i] for c, n, i in zip(self.ctx, new, group)], page, 1)
        shuffle = list(range(pages + count))
        rng.shuffle(shuffle)
        rows = [[shuffle[p] for p in lead[i] if p >= 0] + [shuffle[pages + p] for p in t if p >= 0] for i, t in zip(group, own_table)]
        self.table = [r + [-1] * (max(map(len, rows)) - len(r)) for r in rows]
        self.pages = pages + count
        nan = torch.full((self.pages, kv, page, D), float("nan"))
        self.k, self.v = nan.clone(), nan.clone()
        for b, row in enumerate(self.table):
            for i in range(self.ctx[b] + new[b]):
                self.k[row[i // page], :, i % page] = torch.randn(kv, D, generator=g) / ks
                self.v[row[i // page], :, i % page] = torch.randn(kv, D, generator=g) / vs
        self.k, self.v = self.k.to(cache).cuda(), self.v.to(cache).cuda()
        self.q = (torch.randn(self.cu[-1], heads, D, generator=g) * q_scale).to(dtype).cuda()
        self.masks = None
        if mask == "tree":
            self.masks = [m for n in new for m in _tree_mask(rng, n)]
        elif mask == "random":
            self.masks = [rng.getrandbits(n) if i % 3 else 0 for n in new for i in range(n)]

    def args(self):
        words = max(1, -(-max(self.new) // 32))
        return ((self.q, self.k, self.v, _ints(self.table), _ints(self.cu), _ints(self.ctx), _ints(self.first), _ints(self.shared)),
                dict(mask=None if self.masks is None else _words(self.masks, words), max_new=max(self.new), k_scale=self.ks, v_scale=self.vs))

    def run(self, **kw):
        import paged
        a, k = self.args()
        return paged.shared_attention(*a, **{**k, **kw})

    def check(self, got=None, scale=None, **kw):
        got = self.run(scale=scale, **kw) if got is None else got
        want, spread = R.attention(self.q.double().cpu(), self.k.float().double().cpu() * self.ks, self.v.float().double().cpu() * self.vs,
                                   self.table, self.cu, self.ctx, self.page, self.masks, scale)
        g = got.double().cpu()
        lim = HALF[self.dtype] * (want.abs() + spread) + 4e-5 * spread + 1e-7
        assert not g.isnan().any()
        assert ((g - want).abs() <= lim).all(), ((g - want).abs() / lim).max()
        return got


@pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, BF16), (F16, E4), (BF16, E4)])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_decode_step(cuda, D, dtype, cache):
    e4 = cache == E4
    Case(D, 8, 2, D, 16, [3, 2], [200, 64], [0, 5, 70, 31, 0], [1] * 5, dtype, cache, ks=0.0625 if e4 else 1.0, vs=0.3 if e4 else 1.0).check()


@pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, E4)])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_trees_of_many_rows(cuda, D, dtype, cache):
    Case(D + 1, 8, 2, D, 32, [4], [300], [0, 70, 13, 1], [13, 40, 1, 22], dtype, cache, "tree").check()


@pytest.mark.parametrize("heads,kv", [(32, 32), (32, 8), (16, 2), (12, 4), (8, 1), (5, 1), (34, 2), (3, 3), (64, 1)])
@pytest.mark.parametrize("n", [1, 3, 21])
def test_head_groups(cuda, heads, kv, n):
    Case(heads + n, heads, kv, 64, 16, [2, 3], [90, 33], [50, 7, 0, 1, 16], [n, max(1, n - 2), 1, n, 2], mask="tree").check()


@pytest.mark.parametrize("page", [1, 2, 8, 16, 32, 64, 128, 256])
def test_page_sizes(cuda, page):
    Case(page, 4, 1, 128, page, [2, 2], [260, 127], [0, 130, 64, 3], [3, 2, 1, 5], mask="tree").check()


@pytest.mark.parametrize("D", [8, 40, 112, 248])
def test_other_head_sizes(cuda, D):
    Case(D, 6, 2, D, 16, [2], [48], [33, 0], [4, 9], mask="tree").check()


@pytest.mark.parametrize("members", [1, 2, 7, 40, 130])
def test_sizes_of_groups(cuda, members):
    rng = random.Random(members)
    Case(members, 8, 2, 64, 16, [members, 2], [161, 40], [rng.randrange(40) for _ in range(members + 2)], [1] * (members + 2)).check()


@pytest.mark.parametrize("groups", [1, 60, 299])
def test_more_sequences_than_the_plan_has_threads(cuda, groups):
    rng = random.Random(groups)
    sizes = [600 // groups // 2 if groups < 299 else 2] * groups
    n = sum(sizes)
    Case(groups, 4, 2, 64, 16, sizes, [rng.randrange(16, 80) for _ in sizes], [rng.randrange(20) for _ in range(n)],
         [1 if i % 7 else 0 for i in range(n)]).check()


def test_chunks_of_prompts(cuda):
    """A chain of many new tokens: tiles of 128 rows over the shared rows and over the rest."""
    Case(3, 8, 2, 128, 16, [3], [333], [20, 0, 150], [130, 64, 40], BF16).check()


def test_masks_that_leave_rows_empty(cuda):
    Case(4, 4, 2, 64, 16, [2, 2], [0, 64], [0, 0, 0, 5], [33, 7, 12, 2], mask="random").check()


def test_large_scores_and_scales(cuda):
    Case(5, 8, 2, 128, 16, [4], [500], [3, 60, 0, 9], [1, 2, 1, 1], q_scale=6.0).check(scale=0.3)
    Case(6, 8, 2, 64, 16, [4], [500], [3, 60, 0, 9], [1, 2, 1, 1]).check(scale=-0.2)


def test_long_prefix(cuda):
    """More ranges than one, of shared rows and of a sequence's own."""
    Case(7, 16, 2, 128, 16, [6], [9000], [2500, 0, 1, 700, 64, 8], [1, 1, 2, 1, 3, 1]).check()


@pytest.mark.parametrize("dtype,cache,D", [(F16, F16, 128), (BF16, E4, 64), (F16, F16, 256)])
def test_wide_tables(cuda, dtype, cache, D):
    """By the table's width the call may be a large one: each part has a launch of its own where their kernels differ."""
    import paged
    c = Case(20, 16, 2, D, 16, [9, 4], [700, 90], [50, 0, 1, 70, 64, 8, 3, 16, 31, 2, 0, 40, 5], [1] * 13, dtype, cache)
    a, k = c.args()
    wide = torch.full((13, 12000), -1, dtype=torch.int32, device="cuda")
    wide[:, :a[3].shape[1]] = a[3]
    assert 13 * 16 * 12000 * 16 > 3 << 23
    c.check(paged.shared_attention(*a[:3], wide, *a[4:], **k))
    c.check()


def test_sequences_outside_groups_and_empty_groups(cuda):
    import paged
    c = Case(8, 8, 2, 64, 16, [2, 3, 2], [100, 50, 200], [4, 0, 7, 9, 60, 33, 2], [1, 2, 1, 1, 3, 1, 1])
    a, k = c.args()
    first, shared = [2, 2, 5, 5], [77, 48, 16]  # the first two and the last two sequences stand alone; two groups are empty
    c.check(paged.shared_attention(*a[:6], _ints(first), _ints(shared), **k))
    c.check(paged.shared_attention(*a[:6], _ints([0]), _ints([]), **k))


def test_shared_rows_past_a_context_and_odd_counts(cuda):
    """More rows than a member has cached, negative ones, and counts that are no whole blocks."""
    import paged
    c = Case(9, 8, 2, 64, 16, [3, 2], [96, 48], [0, 11, 40, 0, 3], [1, 2, 1, 1, 1])
    a, k = c.args()
    # the tables agree for 96 and 48 rows; no member of a group has fewer cached
    for shared in ([10 ** 9, 10 ** 9], [96, 0], [95, -7], [17, 33], [2 ** 31 - 1, 1]):
        c.check(paged.shared_attention(*a[:7], _ints(shared), **k))


def test_groups_that_descend_stay_in_bounds(cuda):
    """No meaning, but nothing outside the tensors is touched, and sequences outside keep their results."""
    import paged
    c = Case(10, 8, 2, 64, 16, [4, 2], [64, 32], [0, 11, 40, 0, 3, 5], [1, 2, 1, 1, 1, 1])
    a, k = c.args()
    out = paged.shared_attention(*a[:6], _ints([0, 4, -3, 99]), _ints([64, 32, 32]), **k)
    c.check(out)  # the starts count as 0, 4, 4, 6: the last group shares 32 rows


def test_missing_pages_and_padding(cuda):
    """Rows of pages outside the pool are not seen, shared or not; tokens of no sequence keep their rows."""
    import paged
    c = Case(11, 8, 2, 64, 16, [3], [128], [20, 40, 0], [2, 1, 1])
    for row in c.table:
        row[3] = -1
    c.table[1][9] = 10 ** 6
    c.check()
    c.cu = [x + 2 for x in c.cu]
    c.q = torch.cat([c.q[:2], c.q, c.q[:1]])
    a, k = c.args()
    out = torch.full_like(c.q, 7.0)
    paged.shared_attention(*a, **k, out=out)
    assert (out[:2] == 7).all() and (out[-1] == 7).all() and (out[2:-1] != 7).any()


def test_what_nobody_sees_may_hold_anything(cuda):
    """NaN behind a sequence's rows (Case), infinite values in a masked new row."""
    c = Case(12, 8, 2, 64, 16, [2], [64], [3, 30], [2, 4], mask="tree")
    c.masks = [1, 2] + [1, 1 | 2, 1 | 4, 1 | 8]
    b, row = 1, c.ctx[1] + 2  # node 2 of the second tree: seen by itself alone
    for x in (c.k, c.v):
        x[c.table[b][row // 16], :, row % 16] = float("inf")
    a, k = c.args()
    import paged
    out = paged.shared_attention(*a, **k)
    # Every other token is within the tolerance of what it would be without.  Not to the bit: rows that an infinite value has made NaN
    # are summed up again in another order and with weights that are not rounded.
    c.k, c.v = c.k.nan_to_num(posinf=0.0), c.v.nan_to_num(posinf=0.0)
    out[4] = c.run()[4]
    c.check(out)


def test_repeats_to_the_bit_and_other_streams(cuda):
    import paged
    c = Case(13, 16, 2, 128, 16, [9, 3], [1500, 700], list(range(0, 240, 20)), [1] * 12)
    a, k = c.args()
    first = c.check()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        other = paged.shared_attention(*a, **k, stream=s)
        s.synchronize()
        assert torch.equal(first, other)


def test_captured(cuda):
    """Replays follow the index tensors; eager calls between them keep their results."""
    import paged
    c = Case(14, 16, 2, 128, 16, [5, 4], [800, 320], [3, 90, 0, 16, 33, 1, 2, 64, 5], [1] * 9)
    a, k = c.args()
    out = torch.empty_like(c.q)
    paged.shared_attention(*a, **k, out=out)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        paged.shared_attention(*a, **k, out=out)
    for shared in ([800, 320], [0, 160], [512, 0]):
        a[7].copy_(_ints(shared))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        assert torch.equal(replayed, paged.shared_attention(*a, **k))
        c.check(replayed)


def test_refusals(cuda):
    import paged
    c = Case(15, 4, 2, 64, 16, [2], [32], [0, 1], [1, 1])
    a, k = c.args()
    for i, bad in ((6, a[6].long()), (6, a[6][:1]), (6, a[6].cpu()), (7, a[7].float()), (7, a[7].cpu()), (7, a[7][None]), (0, a[0].float())):
        with pytest.raises(ValueError):
            paged.shared_attention(*a[:i], bad, *a[i + 1:], **k)
