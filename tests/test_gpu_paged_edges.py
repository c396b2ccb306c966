"""GPU tests of the paged calls' far ends: tables with room for more rows than 32 bits count, paths with entries that
are no nodes, arguments that vanish in 32 bits or look strided,
indices out of every range."""

import random

import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("n", [600, 1100])
def test_attention_with_a_table_of_more_than_2_to_the_30_rows(cuda, n):
    """Small heads (the vector-ALU kernel), so many query rows that the length of a range passes every 32-bit number."""
    import paged
    ctx, heads, D, page, width = 100, 8, 8, 65536, 16400
    g = torch.Generator().manual_seed(n)
    k, v = (torch.randn(1, 1, page, D, generator=g).half() for _ in range(2))
    q = torch.randn(n, heads, D, generator=g).half()
    table = [[0] + [-1] * (width - 1)]
    assert width * page > 2 ** 30
    got = paged.tree_attention(q.cuda(), k.cuda(), v.cuda(), _ints(table), _ints([0, n]), _ints([ctx])).double().cpu()
    want, spread = R.attention(q.double(), k.double(), v.double(), [table[0][:1]], [0, n], [ctx], page)
    # the output's rounding, and fp32 scores and sums
    assert ((got - want).abs() <= 2.0 ** -11 * want.abs() + 4e-5 * spread + 1e-7).all()


@pytest.mark.parametrize("path", [[0, 2, 20, -5, 4, 18], [-1] + list(range(12)), [-1, -1, 3, 5, 9, -7, 11, 99, 12, 13, 14, 15, 19],
                                  [-1] * 70 + [1, 4, 6, -1, 7] + [-1] * 60 + [8, 15]], ids=lambda p: str(len(p)))
def test_commit_path_closes_up_over_skipped_entries(cuda, path):
    """The k-th entry that is a node becomes row ctx + k, so that `lens` counts the rows that were kept."""
    import paged
    ctx, n, page = 13, 20, 16
    table = [2, 0, 1]
    k, v = (torch.randn(2, 3, 2, page, 64, device="cuda").half() for _ in range(2))
    want = [k.clone(), v.clone()]
    nodes = [p for p in path if 0 <= p < n]
    for w, src in zip(want, (k.clone(), v.clone())):
        for j, node in enumerate(nodes):
            d, s = ctx + j, ctx + node
            w[:, table[d // page], :, d % page] = src[:, table[s // page], :, s % page]
    lens = paged.commit_path(k, v, _ints([table]), _ints([0, n]), _ints([ctx]), _ints([path]))
    assert lens.tolist() == [ctx + len(nodes)]
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_commit_path_of_many_skipped_entries(cuda):
    import paged
    rng = random.Random(5)
    B, n, page = 6, 200, 32
    k = torch.randn(1, 8 * B, 1, page, 64, device="cuda").half()
    table = [list(range(8 * b, 8 * b + 8)) for b in range(B)]
    ctx = [rng.randint(0, 50) for _ in range(B)]
    paths = [[x for node in sorted(rng.sample(range(n), 90)) for x in ([node] if rng.random() < 0.6 else [-1, node])][:100] for _ in range(B)]
    paths = [p + [-1] * (100 - len(p)) for p in paths]
    want = k.clone()
    for b, p in enumerate(paths):
        for j, node in enumerate(x for x in p if x >= 0):
            d, s = ctx[b] + j, ctx[b] + node
            want[:, table[b][d // page], :, d % page] = k[:, table[b][s // page], :, s % page]
    v = k.clone()
    lens = paged.commit_path(k, v, _ints(table), _ints([n * b for b in range(B + 1)]), _ints(ctx), _ints(paths))
    assert lens.tolist() == [c + sum(x >= 0 for x in p) for c, p in zip(ctx, paths)]
    assert torch.equal(k, want) and torch.equal(v, want)


def _small(**kw):
    args = dict(q=torch.ones(1, 2, 64, device="cuda").half(), k_cache=torch.ones(2, 1, 16, 64, device="cuda").half(),
                v_cache=torch.ones(2, 1, 16, 64, device="cuda").half(), table=_ints([[0, 1]]), cu=_ints([0, 1]), ctx=_ints([17]))
    args.update(kw)
    return args


@pytest.mark.parametrize("scale", [1e-50, -1e-60])
def test_a_scale_that_fp32_has_as_zero_is_refused(cuda, scale):
    """It must not become the default of 1 / sqrt(head_dim)."""
    import paged
    with pytest.raises(ValueError, match="scale"):
        paged.tree_attention(**_small(scale=scale))


def test_single_entries_of_wider_tensors(cuda):
    """One entry is contiguous whatever its stride says."""
    import paged
    a = _small()
    want = paged.tree_attention(**a)
    wide = torch.zeros(1, 7, dtype=torch.int32, device="cuda")
    wide[0, 3] = 17
    assert wide[:, 3].stride(0) != 1
    assert torch.equal(paged.tree_attention(**_small(ctx=wide[:, 3])), want)
    narrow = torch.zeros(1, 2, 5, dtype=torch.int32, device="cuda")[:, :1, 4]
    assert narrow.shape == (1, 1) and narrow.stride(1) != 1
    one = paged.tree_attention(**_small(ctx=_ints([3]), table=_ints([[0]])))
    assert torch.equal(paged.tree_attention(**_small(ctx=_ints([3]), table=narrow)), one)


@pytest.mark.parametrize("first,last", [(-2 ** 31, 3), (-5, 3), (-2 ** 31, -2 ** 31), (2 ** 31 - 1, 2 ** 31 - 1), (0, 2 ** 31 - 1)])
@pytest.mark.parametrize("ctx", [2 ** 31 - 1, -2 ** 31, 14])
def test_indices_of_any_value_stay_within_table_and_pool(cuda, first, last, ctx):
    """Ends of the new tokens and lengths that no call should have: what is written is a token's own row, or nothing."""
    import beam
    import paged
    page, D = 16, 64
    kc, vc = (torch.full((3, 1, page, D), 7.0, device="cuda").half() for _ in range(2))
    table, cu, c = _ints([[2, 0]]), _ints([first, last]), _ints([ctx])
    x = torch.arange(1, 4, device="cuda").half()[:, None, None].expand(3, 1, D).contiguous()
    paged.append(x, x, kc, vc, table, cu, c, rotary_dim=0)
    want = torch.full((3, 1, page, D), 7.0).half()
    if first <= 0 < last and ctx <= 14:
        for i in range(3):
            row = max(ctx, 0) + i
            want[[2, 0][row // page], 0, row % page] = i + 1
    assert torch.equal(kc.cpu(), want) and torch.equal(vc.cpu(), want)
    paged.tree_attention(x, kc, vc, table, cu, c)
    before = kc.clone()
    lens = paged.commit_path(kc[None], vc[None], table, cu, c, _ints([[2 ** 31 - 2, 2 ** 30, -7]]))
    assert torch.equal(kc, before) and torch.equal(vc, before) and lens.shape == (1,)
    beam.reorder(kc[None], vc[None], table, c, _ints([[-2 ** 31]]), _ints([[2 ** 31 - 1]]))
    assert torch.equal(kc, before) and torch.equal(vc, before)
