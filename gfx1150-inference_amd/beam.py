"""Beam search over a paged key/value cache: the selection of a step and the reordering that follows it.

A step of ``beams`` hypotheses for each sentence: ``select`` picks the best continuations from the logits, and
``reorder`` lets every sequence continue its parent's cache.  Full pages are shared, only the open page is
copied, into a page that the caller provides.  See ``paged`` for the cache's tensors.
"""

from __future__ import annotations

import paged
import paged_module as _ops


def select(logits, scores, stream=None):
    """``(scores, parents, tokens)``, each ``[sentences, beams]`` (float32, int32, int32), of the best
    ``beams`` totals ``scores[s, w] + log_softmax(logits[s, w])`` of each sentence in descending order; equal
    totals go to the lower beam, then the lower token.  Totals are formed in 64 bits; where a score's size makes
    those of a beam's different logits equal (-1e30), the larger logit is the better one.

    ``logits`` ``[sentences, beams, vocab]`` float32, float16 or bfloat16 (vocab contiguous), ``scores``
    ``[sentences, beams]`` float32.  The first step of a search gives all beams but one a score of -inf.  A
    total that is not a number counts as -inf: all of a beam's where a logit is NaN or +inf."""
    return paged._on(stream, _ops.beam_select, logits, scores)


def reorder(k_cache, v_cache, table, lens, parents, fresh, stream=None):
    """``(table, lens)`` of the sequences after a step, for sequences ``s * beams + w`` that continue
    ``parents[s, w]``: the parent's length, its full pages shared, and page ``fresh[s, w]`` as the open page, into
    which the rows of the parent's open page are copied in every layer of ``k_cache`` and ``v_cache``
    ``[layers, pages, kv_heads, page_size, head_dim]``.

    ``table`` ``[sentences * beams, width]`` and ``lens`` ``[sentences * beams]`` describe the sequences before the
    step; ``parents`` and ``fresh`` are contiguous int32 ``[sentences, beams]``.  No fresh page may be in use by a
    sequence of ``table``; the parents' open pages are free afterwards."""
    return paged._on(stream, _ops.beam_reorder, k_cache, v_cache, table, lens, parents, fresh)
