"""GPU test of paged.tree_attention's plan over thousands of sequences; tolerances and restatement as in
test_gpu_paged_attention.py."""

import pytest

from test_gpu_paged_attention import Case

pytestmark = pytest.mark.gpu


def test_thousands_of_sequences(cuda):
    """The plan goes over the sequences 64 at a time, some three hundred times; a few are long enough to be cut."""
    B = 20000
    ctx = [i % 3 for i in range(B)]
    ctx[7], ctx[9000], ctx[B - 1] = 700, 3000, 1500
    Case(58, 2, 1, 64, 16, ctx, [1] * B, mask=None).check()
