"""CPU tests of what qmm_paged_evict refuses of its outputs' strides (pointers here are never dereferenced)."""

import pytest

from test_paged_contexts_host import _evict
from test_paged_host import L, _kv, _refused

# two layers, three sequences, two kv heads of 64 rows
SHAPE = dict(num_layers=2, batch=3, kv_heads=2)
APART = dict(wo_layer=384, wo_batch=128, wo_head=64)


@pytest.mark.parametrize("strides", [dict(wo_layer=0), dict(wo_batch=0), dict(wo_head=0), dict(wo_head=63), dict(wo_batch=127), dict(wo_layer=383),
                                     dict(wo_layer=-384), dict(wo_batch=64), dict(wo_layer=128)], ids=lambda s: str(s))
def test_weights_that_overlap_are_refused(strides):
    """Weights of several layers, sequences or heads in one place, which workgroups would write in any order."""
    _refused(L.qmm_paged_evict(_kv(**SHAPE), _evict(**{**APART, **strides}), None, 0, None), "overlap")
    assert L.qmm_paged_evict_workspace(_kv(**SHAPE), _evict(**{**APART, **strides})) == 0


@pytest.mark.parametrize("strides", [dict(), dict(wo_head=192, wo_batch=64), dict(wo_layer=64, wo_batch=256, wo_head=128), dict(wo_layer=1 << 40),
                                     dict(w_layer=0, w_batch=0, w_head=0)], ids=lambda s: str(s))
def test_other_orders_and_expanded_inputs_are_taken(strides):
    assert L.qmm_paged_evict_workspace(_kv(**SHAPE), _evict(**{**APART, **strides})) > 0


def test_an_axis_of_one_needs_no_stride():
    assert L.qmm_paged_evict_workspace(_kv(num_layers=1, batch=1, kv_heads=1), _evict(wo_layer=0, wo_batch=0, wo_head=0)) > 0
