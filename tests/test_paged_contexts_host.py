"""CPU tests of the normed append, the shared-prefix and the weighted attention and the eviction: the ctypes mirrors match
the C structures, and every refusal comes before any GPU work (pointers here are never dereferenced)."""

import ctypes
import os
import subprocess

import pytest

import paged
import qmm
from test_paged_host import BAD_KV, L, P, _kv, _new, _query, _refused


def _fill(c, kw):
    for k, v in kw.items():
        setattr(c, k, v)
    return ctypes.byref(c)


def _norm(**kw):
    return _fill(qmm.PagedNorm(q_weight=P, k_weight=P, axes=None, axis_stride=0, weight_dtype=qmm.DTYPE_F16, num_axes=0, eps=1e-6), kw)


def _groups(**kw):
    return _fill(qmm.PagedGroups(first=P, shared=P, count=1), kw)


def _weights(**kw):
    return _fill(qmm.PagedWeights(old_sums=P, new_sums=P, old_batch=128, old_head=64, new_batch=128, new_head=64, rows=64), kw)


def _evict(**kw):
    return _fill(qmm.PagedEvict(weights=P, weights_out=2 * P, fresh=P, table_out=2 * P, lens_out=2 * P, w_layer=256, w_batch=128, w_head=64,
                                wo_layer=256, wo_batch=128, wo_head=64, fresh_stride=2, rows=64, fresh_width=2, keep=30, recent=4, sinks=1), kw)


def test_structures_match_the_header(tmp_path):
    names = {"qmm_paged_norm": qmm.PagedNorm, "qmm_paged_groups": qmm.PagedGroups, "qmm_paged_weights": qmm.PagedWeights,
             "qmm_paged_evict_args": qmm.PagedEvict}
    lines = ['#include "qmm.h"', "#include <stdio.h>", "int main(void) {"]
    for c, m in names.items():
        lines += [f'printf("%zu\\n", offsetof({c}, {f[0]}));' for f in m._fields_] + [f'printf("%zu\\n", sizeof({c}));']
    src = tmp_path / "s.c"
    src.write_text("\n".join(lines + ["return 0; }"]))
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-I" + include, str(src), "-o", str(tmp_path / "s")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for m in names.values():
        want += [getattr(m, f[0]).offset for f in m._fields_] + [ctypes.sizeof(m)]
    assert got == want


@pytest.mark.parametrize("bad", BAD_KV, ids=lambda b: str(b))
def test_cache_refusals(bad):
    kv = _kv(**bad)
    _refused(L.qmm_paged_append_normed(kv, _new(), _norm(), None))
    _refused(L.qmm_paged_shared_attention(kv, _query(), _groups(), None, 0, None))
    _refused(L.qmm_paged_weighted_attention(kv, _query(), _weights(), None, 0, None))
    _refused(L.qmm_paged_evict(kv, _evict(), None, 0, None))
    assert L.qmm_paged_shared_workspace(kv, _query(), _groups()) == 0
    assert L.qmm_paged_weighted_workspace(kv, _query(), _weights()) == 0
    assert L.qmm_paged_evict_workspace(kv, _evict()) == 0


def test_missing_structures():
    _refused(L.qmm_paged_append_normed(_kv(), _new(), None, None), "norm")
    _refused(L.qmm_paged_append_normed(_kv(), None, _norm(), None), "in")
    _refused(L.qmm_paged_shared_attention(_kv(), _query(), None, None, 0, None), "groups")
    _refused(L.qmm_paged_weighted_attention(_kv(), _query(), None, None, 0, None), "weights")
    _refused(L.qmm_paged_evict(_kv(), None, None, 0, None), "args")
    _refused(L.qmm_paged_evict(None, _evict(), None, 0, None), "kv")


@pytest.mark.parametrize("bad", [dict(weight_dtype=qmm.DTYPE_BF16), dict(weight_dtype=qmm.DTYPE_E4M3), dict(eps=-1e-6), dict(eps=float("nan")),
                                 dict(eps=float("inf")), dict(q_weight=P + 1), dict(weight_dtype=qmm.DTYPE_F32, k_weight=P + 2)], ids=lambda b: str(b))
def test_norm_refusals(bad):
    _refused(L.qmm_paged_append_normed(_kv(), _new(), _norm(**bad), None))


def test_axes_refusals():
    axes = (ctypes.c_uint8 * 32)(*[i % 3 for i in range(32)])
    at = ctypes.addressof(axes)
    _refused(L.qmm_paged_append_normed(_kv(), _new(), _norm(axes=at, num_axes=3), None), "positions")
    _refused(L.qmm_paged_append_normed(_kv(), _new(positions=P), _norm(axes=at, num_axes=2), None), "below")
    _refused(L.qmm_paged_append_normed(_kv(), _new(positions=P), _norm(axes=at, num_axes=0), None), "num_axes")
    _refused(L.qmm_paged_append_normed(_kv(), _new(positions=P, freq_base=0.0), _norm(axes=at, num_axes=3), None), "freq_base")


@pytest.mark.parametrize("bad", [dict(count=-1), dict(count=70000), dict(first=None), dict(shared=None)], ids=lambda b: str(b))
def test_group_refusals(bad):
    _refused(L.qmm_paged_shared_attention(_kv(), _query(), _groups(**bad), None, 0, None))
    assert L.qmm_paged_shared_workspace(_kv(), _query(), _groups(**bad)) == 0


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(old_sums=None), dict(new_sums=None), dict(old_sums=P + 2), dict(new_batch=256), dict(new_head=32)],
                         ids=lambda b: str(b))
def test_sums_refusals(bad):
    _refused(L.qmm_paged_weighted_attention(_kv(), _query(), _weights(**bad), None, 0, None))
    assert L.qmm_paged_weighted_workspace(_kv(), _query(), _weights(**bad)) == 0


@pytest.mark.parametrize("strides", [dict(new_batch=0), dict(new_head=0), dict(new_head=63), dict(new_batch=100), dict(new_batch=-128)], ids=lambda b: str(b))
def test_sums_that_overlap_are_refused(strides):
    """Sums of several heads or sequences in one place, as of an expanded tensor; as an input they are fine."""
    _refused(L.qmm_paged_weighted_attention(_kv(), _query(), _weights(old_sums=2 * P, **strides), None, 0, None), "overlap")
    assert L.qmm_paged_weighted_workspace(_kv(), _query(), _weights(old_sums=2 * P, old_batch=0, old_head=0)) > 0
    assert L.qmm_paged_weighted_workspace(_kv(), _query(), _weights(old_sums=2 * P, new_batch=64, new_head=128)) > 0


@pytest.mark.parametrize("bad", [dict(dtype=qmm.DTYPE_E4M3), dict(heads=3), dict(q=None), dict(scale=float("nan"))], ids=lambda b: str(b))
def test_query_refusals(bad):
    _refused(L.qmm_paged_shared_attention(_kv(), _query(**bad), _groups(), None, 0, None))
    _refused(L.qmm_paged_weighted_attention(_kv(), _query(**bad), _weights(), None, 0, None))


@pytest.mark.parametrize("bad", [dict(keep=0), dict(recent=-1), dict(sinks=-1), dict(recent=30), dict(rows=-1), dict(fresh_width=1), dict(fresh_width=-1),
                                 dict(weights=None), dict(weights_out=None), dict(weights_out=P), dict(weights=P + 2), dict(fresh=None),
                                 dict(table_out=None), dict(table_out=P), dict(lens_out=None), dict(lens_out=P)], ids=lambda b: str(b))
def test_evict_refusals(bad):
    _refused(L.qmm_paged_evict(_kv(), _evict(**bad), None, 0, None))
    assert L.qmm_paged_evict_workspace(_kv(), _evict(**bad)) == 0


def test_evict_counts_are_bounded():
    _refused(L.qmm_paged_evict(_kv(batch=40000), _evict(), None, 0, None), "too many")


def test_workspaces_are_checked():
    kv, q = _kv(table_width=4096), _query()
    for need, call in ((L.qmm_paged_shared_workspace(kv, q, _groups()), lambda w, n: L.qmm_paged_shared_attention(kv, q, _groups(), w, n, None)),
                       (L.qmm_paged_weighted_workspace(kv, q, _weights()), lambda w, n: L.qmm_paged_weighted_attention(kv, q, _weights(), w, n, None)),
                       (L.qmm_paged_evict_workspace(kv, _evict()), lambda w, n: L.qmm_paged_evict(kv, _evict(), w, n, None))):
        assert need > 0
        _refused(call(P, need - 1), "workspace")
        _refused(call(P + 8, need), "workspace")


def test_nothing_to_do_is_accepted():
    assert L.qmm_paged_append_normed(_kv(), _new(tokens=0), _norm(), None) == qmm.QMM_OK
    assert L.qmm_paged_append_normed(_kv(batch=0), _new(), _norm(), None) == qmm.QMM_OK
    assert L.qmm_paged_shared_attention(_kv(), _query(tokens=0), _groups(), None, 0, None) == qmm.QMM_OK
    assert L.qmm_paged_shared_attention(_kv(batch=0), _query(), _groups(), None, 0, None) == qmm.QMM_OK
    assert L.qmm_paged_weighted_attention(_kv(batch=0), _query(), _weights(), None, 0, None) == qmm.QMM_OK
    assert L.qmm_paged_weighted_attention(_kv(), _query(tokens=0), _weights(rows=0), None, 0, None) == qmm.QMM_OK
    assert L.qmm_paged_evict(_kv(batch=0), _evict(), None, 0, None) == qmm.QMM_OK


def test_python_refuses_cpu_tensors():
    import torch
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    c, x, w = torch.zeros(4, 2, 16, 64, dtype=torch.float16), torch.zeros(1, 2, 64, dtype=torch.float16), torch.zeros(1, 2, 64)
    for call in (lambda: paged.append(x, x, c, c, i(1, 4), i(2), i(1), k_norm=w[0, 0]),
                 lambda: paged.shared_attention(x, c, c, i(1, 4), i(2), i(1), i(2), i(1)),
                 lambda: paged.weighted_attention(x, c, c, i(1, 4), i(2), i(1), w),
                 lambda: paged.evict(c[None], c[None], i(1, 4), i(1), w[None], i(1, 2), 20)):
        with pytest.raises(ValueError, match="GPU"):
            call()
