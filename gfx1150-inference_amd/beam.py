"""Beam search over a paged key/value cache: the selection of a step and the reordering that follows it.

A step of ``beams`` hypotheses for each sentence: ``select`` picks the best continuations from the logits, and
``reorder`` lets every sequence continue its parent's cache.  Full pages are shared, only the open page is
copied, into a page that the caller provides.  See ``paged`` for the cache's tensors.
"""

from __future__ import annotations

import torch

import paged
import qmm

_lib = qmm.lib()


def select(logits, scores, stream=None):
    """``(scores, parents, tokens)``, each ``[sentences, beams]`` (float32, int32, int32), of the best
    ``beams`` totals ``scores[s, w] + log_softmax(logits[s, w])`` of each sentence in descending order; equal
    totals go to the lower beam, then the lower token.

    ``logits`` ``[sentences, beams, vocab]`` float32, float16 or bfloat16 (vocab contiguous), ``scores``
    ``[sentences, beams]`` float32.  The first step of a search gives all beams but one a score of -inf.  A
    total that is not a number counts as -inf."""
    if not logits.is_cuda or logits.dim() != 3:
        raise ValueError("logits must be a [sentences, beams, vocab] tensor on a GPU")
    sentences, beams, vocab = logits.shape
    code = paged._CODE.get(logits.dtype)
    if code is None or code == qmm.DTYPE_E4M3:
        raise ValueError("logits must be float32, float16 or bfloat16")
    st = logits.stride()
    if st[2] != 1 and vocab > 1:
        raise ValueError("vocab must be contiguous in logits")
    device = logits.device
    if scores.dtype != torch.float32 or scores.device != device or tuple(scores.shape) != (sentences, beams) or not scores.is_contiguous():
        raise ValueError("scores must be a contiguous float32 [sentences, beams] tensor on the logits' device")
    out = torch.empty((3, sentences, beams), dtype=torch.int32, device=device)
    best, parents, tokens = out.unbind(0)
    best = best.view(torch.float32)
    handle = paged._on(device, stream)
    need = _lib.qmm_beam_select_workspace(code, sentences, beams, vocab)
    space = torch.empty(need, dtype=torch.uint8, device=device)
    paged._made(stream, out, space)
    rc = _lib.qmm_beam_select(logits.data_ptr(), code, st[0], st[1], scores.data_ptr(), sentences, beams, vocab, best.data_ptr(),
                              parents.data_ptr(), tokens.data_ptr(), space.data_ptr(), need, handle)
    if rc:
        qmm.check(rc)
    return best, parents, tokens


def reorder(k_cache, v_cache, table, lens, parents, fresh, stream=None):
    """``(table, lens)`` of the sequences after a step, for sequences ``s * beams + w`` that continue
    ``parents[s, w]``: the parent's length, its full pages shared, and page ``fresh[s, w]`` as the open page, into
    which the rows of the parent's open page are copied in every layer of ``k_cache`` and ``v_cache``
    ``[layers, pages, kv_heads, page_size, head_dim]``.

    ``table`` ``[sentences * beams, width]`` and ``lens`` ``[sentences * beams]`` describe the sequences before the
    step; ``parents`` and ``fresh`` are contiguous int32 ``[sentences, beams]``.  No fresh page may be in use by a
    sequence of ``table``; the parents' open pages are free afterwards."""
    if not parents.is_cuda:
        raise ValueError("parents must be on a GPU")
    kv = paged._kv_bytes(k_cache, v_cache, table, None, lens, 1.0, 1.0, True)
    device = k_cache.device
    paged._ints(parents, "parents", (None, None), device)
    paged._ints(fresh, "fresh", tuple(parents.shape), device)
    beams = parents.shape[1]
    if parents.numel() != lens.shape[0] or not parents.is_contiguous() or not fresh.is_contiguous():
        raise ValueError("parents and fresh must be contiguous and hold one entry per sequence")
    new_table = torch.empty(table.shape, dtype=torch.int32, device=device)
    new_lens = torch.empty(lens.shape, dtype=torch.int32, device=device)
    paged._made(stream, new_table, new_lens)
    rc = _lib.qmm_beam_reorder(kv, parents.data_ptr(), fresh.data_ptr(), beams, new_table.data_ptr(), new_lens.data_ptr(),
                               paged._on(device, stream))
    if rc:
        qmm.check(rc)
    return new_table, new_lens
