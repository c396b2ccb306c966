"""GPU tests of paged.tree_attention against the 64-bit restatement in paged_reference.py.

Tolerance of an output: its own rounding (half a step), the weights' rounding to the queries' type before the second
product (half a step of sum p |v|), and 4e-5 of sum p |v| for fp32 scores up to about 30 (dot products of 256 terms:
1e-5, the exponential's argument: 2^-19)."""

import random

import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu

F16, BF16, E4 = torch.float16, torch.bfloat16, torch.float8_e4m3fn
HALF = {F16: 2.0 ** -11, BF16: 2.0 ** -8}


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _tree_mask(rng, n):
    masks = [1]
    for i in range(1, n):
        masks.append(masks[rng.randrange(max(0, i - 5), i)] | (1 << i))
    return masks[:n]


def _words(masks, words):
    sign = lambda w: w - (1 << 32) if w >> 31 else w  # noqa: E731
    return _ints([[sign((m >> (32 * w)) & 0xFFFFFFFF) for w in range(words)] for m in masks]).reshape(len(masks), words)


class Case:
    def __init__(self, seed, heads, kv, D, page, ctx, new, dtype=F16, cache=None, mask="tree", ks=1.0, vs=1.0, q_scale=1.0):
        rng = random.Random(seed)
        g = torch.Generator().manual_seed(seed)
        cache = cache or dtype
        self.page, self.dtype, self.heads = page, dtype, heads
        self.ctx, self.new = ctx, new
        self.cu = [0]
        for n in new:
            self.cu.append(self.cu[-1] + n)
        self.table, self.pages = R.make_pages(rng, [c + n for c, n in zip(ctx, new)], page, 1)
        # what no sequence holds is NaN
        nan = torch.full((self.pages, kv, page, D), float("nan"))
        self.k, self.v = nan.clone(), nan.clone()
        for b, row in enumerate(self.table):
            for i in range(ctx[b] + new[b]):
                self.k[row[i // page], :, i % page] = torch.randn(kv, D, generator=g) / ks
                self.v[row[i // page], :, i % page] = torch.randn(kv, D, generator=g) / vs
        self.k, self.v = self.k.to(cache).cuda(), self.v.to(cache).cuda()
        self.q = (torch.randn(self.cu[-1], heads, D, generator=g) * q_scale).to(dtype).cuda()
        self.masks = None
        if mask == "tree":
            self.masks = [m for n in new for m in _tree_mask(rng, n)]
        elif mask == "random":
            self.masks = [rng.getrandbits(n) if i % 3 else 0 for n in new for i in range(n)]
        self.ks, self.vs = ks, vs

    def run(self, **kw):
        import paged
        words = max(1, -(-max(self.new) // 32))
        args = dict(mask=None if self.masks is None else _words(self.masks, words), max_new=max(self.new), k_scale=self.ks, v_scale=self.vs)
        args.update(kw)
        return paged.tree_attention(self.q, self.k, self.v, _ints(self.table).reshape(len(self.ctx), -1), _ints(self.cu), _ints(self.ctx), **args)

    def want(self, scale=None):
        return R.attention(self.q.double().cpu(), self.k.float().double().cpu() * self.ks, self.v.float().double().cpu() * self.vs,
                           self.table, self.cu, self.ctx, self.page, self.masks, scale)

    def check(self, scale=None, **kw):
        if scale is not None:
            kw["scale"] = scale
        got = self.run(**kw)
        assert got.dtype == self.dtype
        want, spread = self.want(scale)
        g = got.double().cpu()
        lim = HALF[self.dtype] * (want.abs() + spread) + 4e-5 * spread + 1e-7
        assert not g.isnan().any()
        assert ((g - want).abs() <= lim).all(), ((g - want).abs() / lim).max()
        return got


@pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, BF16), (F16, E4), (BF16, E4)])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_decode_step(cuda, D, dtype, cache):
    Case(D, 8, 2, D, 16, [0, 1, 63, 200], [1, 1, 1, 1], dtype, cache, None).check()


@pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, BF16), (F16, E4), (BF16, E4)])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_trees(cuda, D, dtype, cache):
    Case(D + 1, 8, 2, D, 32, [0, 70, 130], [13, 40, 1], dtype, cache, "tree", ks=0.0625 if cache == E4 else 1.0,
         vs=0.3 if cache == E4 else 1.0).check()


@pytest.mark.parametrize("heads,kv", [(32, 32), (32, 8), (16, 2), (12, 4), (8, 1), (5, 1), (34, 2), (3, 3), (64, 1)])
@pytest.mark.parametrize("n", [1, 3, 21])
def test_head_groups(cuda, heads, kv, n):
    Case(heads + n, heads, kv, 64, 16, [50, 7], [n, max(1, n - 2)], mask="tree").check()


@pytest.mark.parametrize("page", [1, 2, 4, 8, 16, 32, 64, 128, 256])
def test_page_sizes(cuda, page):
    Case(page, 4, 1, 128, page, [0, 127, 130, 64], [33, 2, 1, 5], mask="tree").check()


@pytest.mark.parametrize("D", [8, 40, 80, 112, 136, 192, 248])
def test_other_head_sizes(cuda, D):
    Case(D, 6, 2, D, 16, [33, 0], [4, 9], mask="tree").check()
    Case(D, 6, 2, D, 16, [33, 0], [4, 9], BF16, E4, mask=None).check()


@pytest.mark.parametrize("n", [2, 31, 32, 33, 64, 65, 127, 128, 129, 150])
def test_tree_sizes(cuda, n):
    Case(n, 4, 2, 64, 16, [3, 65], [n, (n + 1) // 2], mask="random").check()


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16), (96, F16), (256, F16)])
def test_chunks_of_a_prompt(cuda, D, dtype):
    """A chain without a mask, from an empty cache and behind a longer one."""
    Case(D, 4, 2, D, 64, [0, 150, 5], [200, 77, 0], dtype, mask=None).check()


def test_long_contexts(cuda):
    """Many ranges of keys, sequences of very different lengths in one call."""
    Case(21, 4, 1, 64, 16, [5000, 3, 1030], [1, 1, 1], mask=None).check()
    Case(22, 2, 1, 128, 64, [3000, 10], [9, 20], BF16, mask="tree").check()


def test_many_sequences(cuda):
    """More sequences than a wave's lanes, of every length."""
    Case(38, 4, 2, 64, 16, [(7 * i) % 97 for i in range(150)], [1 + (i == 9) for i in range(150)], mask=None).check()
    Case(39, 4, 1, 64, 32, [(11 * i) % 60 for i in range(70)], [(5 * i) % 37 for i in range(70)], BF16, mask="tree").check()
    Case(40, 2, 2, 128, 16, [0] * 130 + [3], [0] * 129 + [2, 70], mask=None).check()


def test_whole_sequences_in_one_range(cuda):
    """Enough (sequence, kv head) pairs that 9000 keys are one workgroup's: every sequence the same pages and queries."""
    import paged
    ctx, heads, D, page, B = 8999, 24, 64, 16, 64
    g = torch.Generator().manual_seed(41)
    k, v = (torch.randn(-(-(ctx + 1) // page), heads, page, D, generator=g).half().cuda() for _ in range(2))
    row = torch.randperm(k.shape[0], generator=g)
    q1 = torch.randn(1, heads, D, generator=g).half()
    out = paged.tree_attention(q1.cuda().expand(B, -1, -1), k, v, row.int().cuda()[None].expand(B, -1), _ints(list(range(B + 1))), _ints([ctx] * B),
                               max_new=1)
    assert torch.equal(out, out[:1].expand_as(out))
    kd, vd = (x.double().cpu()[row].transpose(1, 2).reshape(-1, heads, D)[:ctx + 1] for x in (k, v))
    p = torch.softmax((kd * q1[0].double()).sum(-1) / D ** 0.5, 0)
    want, spread = (p[..., None] * vd).sum(0), (p[..., None] * vd.abs()).sum(0)
    assert ((out[0].double().cpu() - want).abs() <= HALF[F16] * (want.abs() + spread) + 4e-5 * spread).all()


def test_large_scores(cuda):
    """Scores of a hundred: the running maximum moves through the whole context."""
    c = Case(23, 4, 1, 64, 16, [700], [5], mask="tree", q_scale=12.0)
    want, spread = c.want()
    g = c.run().double().cpu()
    # fp32 scores up to 200: 200 * 2^-22 of the weights
    assert ((g - want).abs() <= 2.0 ** -11 * (want.abs() + spread) + 2e-4 * spread).all()


def test_scale_and_negative_scale(cuda):
    Case(24, 4, 2, 64, 16, [40], [20], mask="tree").check(scale=0.3)
    Case(25, 4, 2, 128, 16, [40], [2], mask=None).check(scale=-0.1)


def test_rows_that_see_nothing(cuda):
    """No cached rows and an empty mask: zeros; empty sequences between others."""
    c = Case(26, 4, 2, 64, 16, [0, 0, 40, 9], [5, 0, 3, 0], mask="random")
    c.masks[:5] = [0, 0, 3, 0, 16]
    got = c.check()
    assert (got[[0, 1, 3]] == 0).all()


@pytest.mark.parametrize("D,n,heads", [(64, 20, 4), (128, 3, 4), (128, 40, 8), (256, 12, 4), (96, 9, 4)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_unseen_rows_have_no_effect(cuda, D, n, heads, value):
    """NaN and infinities in new rows that some tokens see and others do not reach only the former."""
    c = Case(27, heads, 2, D, 16, [30], [n], mask="tree")
    clean = c.run().clone()
    bad = n - 2  # a late node
    row = 30 + bad
    pg, slot = c.table[0][row // 16], row % 16
    for cache in (c.k, c.v):
        keep = cache[pg, :, slot].clone()
        cache[pg, :, slot] = value
        got = c.run()
        cache[pg, :, slot] = keep
        for t in range(n):
            if not (c.masks[t] >> bad) & 1:
                # the products of other rows may be taken in another way: the same values up to a rounding
                assert (got[t].float() - clean[t].float()).abs().max() <= 2.0 ** -10 * (1 + clean[t].float().abs().max()), t
    # the value of a seen row reaches those that see it
    c.v[pg, :, slot] = value
    got = c.run()
    for t in range(n):
        if (c.masks[t] >> bad) & 1:
            x = got[t].float()
            assert x.isnan().all() if value != value else (x == value).all(), t


def test_infinite_value_of_a_cached_row(cuda):
    c = Case(28, 8, 1, 128, 16, [100], [30], mask="tree")
    c.v[c.table[0][3], :, 5, 7] = float("inf")
    got = c.run().float()
    assert (got[:, :, 7] == float("inf")).all() and got[:, :, :7].isfinite().all() and got[:, :, 8:].isfinite().all()


def test_bad_pages_are_not_seen(cuda):
    """Page ids outside the pool and rows past the table are left out, whatever the mask says."""
    c = Case(29, 4, 2, 64, 16, [40, 50], [6, 3], mask="tree")
    c.table[0][1] = -1
    c.table[1][0] = c.pages + 5
    c.check()
    c = Case(30, 4, 2, 64, 16, [40, 50], [20, 3], mask="tree")
    c.table = [row[:3] for row in c.table]
    c.check()


def test_strided_operands(cuda):
    """Queries out of a fused projection, K and V in one tensor, an output with room between its heads."""
    c = Case(31, 6, 2, 64, 16, [40, 3], [7, 2], mask="tree")
    plain = c.run()
    both = torch.stack([c.k, c.v], 1)
    c.k, c.v = both[:, 0], both[:, 1]
    fused = torch.randn(9, 10, 64, device="cuda").half()
    fused[:, 2:8] = c.q
    c.q = fused[:, 2:8]
    wide = torch.zeros(9, 6, 96, dtype=F16, device="cuda")
    got = c.run(out=wide[..., :64])
    assert torch.equal(got, plain) and (wide[..., 64:] == 0).all()
    buf = torch.empty(c.q.numel() + 1, dtype=F16, device="cuda")
    c.q = buf[1:].view(9, 6, 64).copy_(c.q)
    got = c.run()
    assert (got.float() - plain.float()).abs().max() <= 2.0 ** -9


def test_unaligned_cache(cuda):
    c = Case(32, 4, 2, 64, 16, [40, 3], [7, 2], mask="tree")
    for name in ("k", "v"):
        t = getattr(c, name)
        buf = torch.empty(t.numel() + 1, dtype=F16, device="cuda")
        setattr(c, name, buf[1:].view(t.shape).copy_(t))
    c.check()


def test_no_tokens(cuda):
    c = Case(33, 4, 2, 64, 16, [40, 3], [0, 0], mask=None)
    assert c.run(max_new=0).shape == (0, 4, 64)


def test_without_max_new_and_wide_table(cuda):
    c = Case(34, 4, 2, 64, 16, [40, 3], [7, 2], mask="tree")
    c.check(max_new=None)
    c.table = [row + [-1] * 300 for row in c.table]
    c.check()


def test_other_stream_and_graph(cuda):
    """On a stream given to the call, and captured: replays follow the inputs."""
    c = Case(35, 8, 2, 128, 16, [300, 20], [5, 9], mask="tree")
    plain = c.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = c.run(stream=side)
    torch.cuda.synchronize()
    assert torch.equal(got, plain)
    words = _words(c.masks, 1)
    import paged
    table, cu, ctx = _ints(c.table), _ints(c.cu), _ints(c.ctx)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged.tree_attention(c.q, c.k, c.v, table, cu, ctx, mask=words, max_new=9)
    q0 = c.q.clone()
    for rep in range(3):
        c.q.copy_(q0 * (1 + rep))
        out.fill_(float("nan"))
        eager = paged.tree_attention(c.q, c.k, c.v, table, cu, ctx, mask=words, max_new=9)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), rep


def test_past_32_bit_offsets(cuda):
    """A pool of more than 2^32 elements: pages at its end."""
    kv, D, page = 8, 128, 128
    pages = 2 ** 32 // (kv * D * page) + 3
    pool = torch.zeros(pages, kv, page, D, dtype=F16, device="cuda")
    c = Case(36, 16, kv, D, page, [200], [4], mask="tree")
    for i, p in enumerate(c.table[0]):
        pool[pages - 1 - i] = c.k[p]
    want = c.check()
    old = c.table
    vpool = torch.zeros_like(pool)
    for i, p in enumerate(old[0]):
        vpool[pages - 1 - i] = c.v[p]
    c.k, c.v, c.table = pool, vpool, [[pages - 1 - i for i in range(len(old[0]))]]
    assert torch.equal(c.run(), want)


def test_refusals(cuda):
    import paged
    c = Case(37, 4, 2, 64, 16, [4], [2], mask="tree")
    t, cu, ctx = _ints(c.table), _ints(c.cu), _ints(c.ctx)
    m = _words(c.masks, 1)
    ok = dict(q=c.q, k_cache=c.k, v_cache=c.v, table=t, cu=cu, ctx=ctx, mask=m)
    paged.tree_attention(**ok)
    for change in (dict(q=c.q.float()), dict(q=c.q[0]), dict(q=c.q.bfloat16()), dict(q=c.q[..., :32]), dict(q=c.q[:, :3]),
                   dict(k_cache=c.k[0]), dict(v_cache=c.v.bfloat16()), dict(k_cache=c.k.cpu()), dict(table=t.long()), dict(table=t[0]),
                   dict(cu=cu[:1]), dict(ctx=torch.cat([ctx, ctx])), dict(mask=m.long()), dict(mask=m[:1]), dict(mask=m[:, :0]),
                   dict(scale=0.0), dict(scale=float("inf")), dict(k_scale=2.0), dict(out=c.q[:1]), dict(out=c.q.float()),
                   dict(k_cache=c.k[:, :, :12], v_cache=c.v[:, :, :12]), dict(max_new=-1), dict(table=t.cpu())):
        with pytest.raises(ValueError):
            paged.tree_attention(**{**ok, **change})
