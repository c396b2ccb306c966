"""GPU tests of the paged calls' far ends: tables with room for more rows than 32 bits count."""

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
