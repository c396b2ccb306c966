"""CPU tests of the paged-cache and beam entry points: the ctypes mirrors match the C structures, and every refusal
comes before any GPU work (pointers here are never dereferenced)."""

import ctypes
import os
import subprocess

import pytest

import beam
import paged
import qmm

L = qmm.lib()
P = 4096  # an address that no refusal reads


def _kv(**kw):
    c = qmm.PagedKV(k=P, v=P, table=P, cu=P, ctx=P, table_stride=4, k_layer=0, k_page=2048, k_head=1024, k_slot=64, v_layer=0,
                    v_page=2048, v_head=1024, v_slot=64, table_width=4, batch=2, dtype=qmm.DTYPE_F16, num_layers=1, num_pages=8,
                    kv_heads=2, page_size=16, head_dim=64, k_scale=1.0, v_scale=1.0)
    for k, v in kw.items():
        setattr(c, k, v)
    return ctypes.byref(c)


def _new(**kw):
    c = qmm.PagedNew(k=P, v=P, q=P, q_out=P, positions=None, k_token=128, k_head=64, v_token=128, v_head=64, q_token=256, q_head=64,
                     qo_token=256, qo_head=64, tokens=3, heads=4, dtype=qmm.DTYPE_F16, rotary_dim=64, neox=0, freq_base=1e4)
    for k, v in kw.items():
        setattr(c, k, v)
    return ctypes.byref(c)


def _query(**kw):
    c = qmm.PagedQuery(q=P, out=P, mask=None, q_token=256, q_head=64, out_token=256, out_head=64, mask_stride=0, tokens=3, max_new=3,
                       heads=4, dtype=qmm.DTYPE_F16, mask_words=0, scale=0.0)
    for k, v in kw.items():
        setattr(c, k, v)
    return ctypes.byref(c)


def _refused(rc, text=""):
    assert rc == qmm.QMM_ERR_INVALID_ARGUMENT
    assert text in qmm.last_error(), qmm.last_error()


def test_structures_match_the_header(tmp_path):
    """The ctypes mirrors have the size and the field offsets of include/qmm.h's structures."""
    names = {"qmm_paged_kv": qmm.PagedKV, "qmm_paged_new": qmm.PagedNew, "qmm_paged_query": qmm.PagedQuery}
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


BAD_KV = [dict(dtype=qmm.DTYPE_F32), dict(dtype=7), dict(batch=-1), dict(batch=70000), dict(num_pages=-1), dict(table_width=-1),
          dict(num_layers=0), dict(kv_heads=0), dict(head_dim=0), dict(head_dim=260), dict(head_dim=12), dict(page_size=0),
          dict(page_size=24), dict(k_scale=0.0), dict(v_scale=-1.0), dict(k_scale=float("nan")), dict(v_scale=2.0), dict(k=None),
          dict(v=None), dict(table=None), dict(ctx=None), dict(k=P + 1)]


@pytest.mark.parametrize("bad", BAD_KV, ids=lambda b: str(b))
def test_cache_refusals(bad):
    kv = _kv(**bad)
    _refused(L.qmm_paged_append(kv, _new(), None))
    _refused(L.qmm_paged_tree_attention(kv, _query(), None, 0, None))
    assert L.qmm_paged_attention_workspace(kv, _query()) == 0
    _refused(L.qmm_paged_commit_path(kv, P, 4, 4, P, None))
    _refused(L.qmm_beam_reorder(kv, P, P, 2, P + 64, P + 128, None))


def test_missing_structures():
    _refused(L.qmm_paged_append(None, _new(), None), "kv")
    _refused(L.qmm_paged_append(_kv(), None, None), "in")
    _refused(L.qmm_paged_append(_kv(cu=None), _new(), None), "cu")
    _refused(L.qmm_paged_tree_attention(None, _query(), None, 0, None), "kv")
    _refused(L.qmm_paged_tree_attention(_kv(), None, None, 0, None), "in")


@pytest.mark.parametrize("bad", [dict(dtype=qmm.DTYPE_F32), dict(dtype=qmm.DTYPE_BF16), dict(tokens=-1), dict(heads=-1), dict(heads=0),
                                 dict(q_out=None), dict(k=None), dict(v=None), dict(rotary_dim=-2), dict(rotary_dim=31),
                                 dict(rotary_dim=66), dict(freq_base=0.0), dict(freq_base=float("inf"))], ids=lambda b: str(b))
def test_append_refusals(bad):
    _refused(L.qmm_paged_append(_kv(), _new(**bad), None))


@pytest.mark.parametrize("bad", [dict(dtype=qmm.DTYPE_E4M3), dict(dtype=qmm.DTYPE_BF16), dict(tokens=-1), dict(max_new=-1), dict(heads=0),
                                 dict(heads=3), dict(heads=70000), dict(q=None), dict(out=None), dict(q=P + 1), dict(mask_words=-1),
                                 dict(scale=float("nan"))], ids=lambda b: str(b))
def test_attention_refusals(bad):
    _refused(L.qmm_paged_tree_attention(_kv(), _query(**bad), None, 0, None))


def test_attention_workspace_is_checked():
    kv, q = _kv(table_width=4096), _query()
    need = L.qmm_paged_attention_workspace(kv, q)
    assert need > 0
    _refused(L.qmm_paged_tree_attention(kv, q, P, need - 1, None), "workspace")
    _refused(L.qmm_paged_tree_attention(kv, q, P + 8, need, None), "workspace")


def test_nothing_to_do_is_accepted():
    assert L.qmm_paged_append(_kv(), _new(tokens=0), None) == qmm.QMM_OK
    assert L.qmm_paged_append(_kv(batch=0), _new(), None) == qmm.QMM_OK
    assert L.qmm_paged_tree_attention(_kv(), _query(tokens=0), None, 0, None) == qmm.QMM_OK
    assert L.qmm_paged_commit_path(_kv(batch=0), P, 4, 4, P, None) == qmm.QMM_OK
    assert L.qmm_beam_select(P, qmm.DTYPE_F32, 10, 10, P, 0, 2, 10, P, P, P, None, 0, None) == qmm.QMM_OK


def test_commit_and_reorder_refusals():
    _refused(L.qmm_paged_commit_path(_kv(), None, 4, 4, P, None), "path")
    _refused(L.qmm_paged_commit_path(_kv(), P, 4, 4, None, None), "lens")
    _refused(L.qmm_paged_commit_path(_kv(), P, 4, -1, P, None), "path_len")
    _refused(L.qmm_beam_reorder(_kv(), P, P, 0, P + 64, P + 128, None), "beams")
    _refused(L.qmm_beam_reorder(_kv(), P, P, 3, P + 64, P + 128, None), "beams")
    _refused(L.qmm_beam_reorder(_kv(), None, P, 2, P + 64, P + 128, None), "parents")
    _refused(L.qmm_beam_reorder(_kv(), P, P, 2, P, P + 128, None), "table_out")
    _refused(L.qmm_beam_reorder(_kv(), P, P, 2, P + 64, P, None), "lens_out")


@pytest.mark.parametrize("dtype,B,W,V", [(qmm.DTYPE_E4M3, 1, 2, 10), (qmm.DTYPE_F32, -1, 2, 10), (qmm.DTYPE_F32, 1, 0, 10),
                                         (qmm.DTYPE_F32, 1, 65, 10), (qmm.DTYPE_F32, 1, 2, 0), (qmm.DTYPE_F32, 1, 2, 2 ** 30 + 1),
                                         (qmm.DTYPE_F32, 2000, 64, 10)])
def test_select_refusals(dtype, B, W, V):
    assert L.qmm_beam_select_workspace(dtype, B, W, V) == 0
    _refused(L.qmm_beam_select(P, dtype, V, V, P, B, W, V, P, P, P, P, 1 << 20, None))


def test_select_pointers_and_workspace():
    need = L.qmm_beam_select_workspace(qmm.DTYPE_F16, 2, 4, 1000)
    assert need > 0
    args = [P, qmm.DTYPE_F16, 4000, 1000, P, 2, 4, 1000, P, P, P]
    _refused(L.qmm_beam_select(*args, P, need - 1, None), "workspace")
    _refused(L.qmm_beam_select(*args, P + 4, need, None), "workspace")
    for i in (0, 4, 8, 9, 10):
        _refused(L.qmm_beam_select(*(None if j == i else a for j, a in enumerate(args)), P, need, None), "non-null")
    _refused(L.qmm_beam_select(P + 1, *args[1:], P, need, None), "aligned")


def test_python_refuses_cpu_tensors():
    import torch
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    c, x = torch.zeros(4, 2, 16, 64, dtype=torch.float16), torch.zeros(1, 2, 64, dtype=torch.float16)
    for call in (lambda: paged.append(x, x, c, c, i(1, 4), i(2), i(1)), lambda: paged.tree_attention(x, c, c, i(1, 4), i(2), i(1)),
                 lambda: paged.commit_path(c[None], c[None], i(1, 4), i(2), i(1), i(1, 3)), lambda: beam.select(x, torch.zeros(1, 2)),
                 lambda: beam.reorder(c[None], c[None], i(2, 4), i(2), i(1, 2), i(1, 2))):
        with pytest.raises(ValueError, match="GPU"):
            call()
