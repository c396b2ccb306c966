"""CPU tests: refusals of paged attention that need more than one argument to see."""

import pytest

import qmm
from test_paged_host import _kv, _query, _refused

L = qmm.lib()


@pytest.mark.parametrize("scale,k_scale", [(1e-30, 1e-30), (-1e-25, 1e-20), (1e30, 1e30), (1e-40, 1.0)])
def test_scores_scale_out_of_range(scale, k_scale):
    """A factor of 0 would make masked scores of -inf NaN; one of infinity every score of 0."""
    kv = _kv(dtype=qmm.DTYPE_E4M3, k_scale=k_scale)
    _refused(L.qmm_paged_tree_attention(kv, _query(scale=scale), None, 0, None), "scale")
    assert L.qmm_paged_attention_workspace(kv, _query(scale=scale)) == 0
