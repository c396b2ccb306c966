"""A paged key/value cache: appending new tokens, attention over it, committing drafted tokens, and evicting rows.

For batches of sequences whose rows live in pages of one pool.  The caller owns every tensor:

* a layer's cache is a K and a V tensor ``[pages, kv_heads, page_size, head_dim]`` (float16, bfloat16 or
  float8_e4m3fn; any strides with ``head_dim`` contiguous, so that K and V may share one tensor);
* ``table`` ``[batch, width]`` int32 holds each sequence's page ids, ``ctx`` ``[batch]`` int32 the rows it has;
* ``cu`` ``[batch + 1]`` int32, not descending, delimits the new tokens, which are concatenated: sequence b has
  tokens ``cu[b]`` to ``cu[b + 1] - 1``, and they take its rows ``ctx[b]``, ``ctx[b] + 1``, ...

A decoding step of a model calls, per layer, ``append`` and ``tree_attention``; a step with drafted
tokens ends with one ``commit_path`` over all layers.  ``shared_attention`` stands for it where sequences begin with the
same pages, ``weighted_attention`` where the rows' attention weights are gathered for ``evict``, which cuts the sequences
to the rows of the largest.  Every call is asynchronous on ``stream`` (the
current one by default) and can be captured into a graph.  The indices are read on the device: a row whose
page is outside the table or the pool is not written, copied or seen, and a token that ``cu`` gives to no sequence
(padding) is passed over: its row of ``q_out`` or ``out`` is left as it was, uninitialised in a new tensor.
"""

from __future__ import annotations

import torch

import qmm  # noqa: F401  (loads the library after torch's HIP runtime)
import paged_module as _ops


def _on(stream, call, *args):
    """The call on `stream`, which torch's current one becomes for it: tensors made for the call belong to it."""
    if stream is None:
        return call(*args)
    with torch.cuda.stream(stream):
        return call(*args)


def append(k, v, k_cache, v_cache, table, cu, ctx, q=None, q_out=None, positions=None, freq_base: float = 10000.0,
           rotary_dim=None, neox: bool = False, k_scale: float = 1.0, v_scale: float = 1.0, stream=None, q_norm=None, k_norm=None,
           norm_eps: float = 1e-6, axes=None):
    """Writes new tokens' keys and values ``[tokens, kv_heads, head_dim]`` into their pages, the keys rotated on
    the way, and the rotated queries ``q`` ``[tokens, heads, head_dim]`` into ``q_out`` (a new tensor by default;
    may be ``q``).  Returns ``q_out``.

    The first ``rotary_dim`` dimensions (all by default; 0: none) turn by ``position * freq_base ** (-2 i /
    rotary_dim)``, pairs ``(2i, 2i + 1)``, or ``(i, i + rotary_dim / 2)`` with ``neox``.  A token's position is its
    row in the cache unless ``positions`` ``[tokens]`` int32 says otherwise (the depth of a drafted tree's
    node).  A float8 cache stores ``value / scale``, saturated at 448; the others need a scale of 1.

    ``q_norm`` and ``k_norm`` ``[head_dim]`` (float32, or the tokens' type) norm every query and key head ahead of its rotation:
    ``x * rsqrt(mean(x^2) + norm_eps) * weight``, not rounded in between.  With ``axes``, a sequence of
    ``rotary_dim / 2`` ints, pair i turns by ``positions[axes[i], token]`` of ``positions`` ``[axes, tokens]``: time, height and
    width of an image's or a video's tokens, in runs of pairs or in turn (a text's token has the same position on
    all)."""
    args = (k, v, k_cache, v_cache, table, cu, ctx, q, q_out, positions, freq_base, rotary_dim, neox, k_scale, v_scale)
    if q_norm is None and k_norm is None and axes is None:
        return _on(stream, _ops.append, *args)
    return _on(stream, _ops.append_normed, *args, q_norm, k_norm, norm_eps, axes)


def tree_attention(q, k_cache, v_cache, table, cu, ctx, mask=None, max_new=None, scale=None, k_scale: float = 1.0,
                   v_scale: float = 1.0, out=None, stream=None):
    """Attention of the new tokens' queries ``[tokens, heads, head_dim]`` (rotated, and their keys and values
    appended) over the cache.  Returns ``out``, alike.

    Token i of a sequence sees the sequence's ``ctx`` cached rows and, of its new tokens j, those with bit
    ``j % 32`` of ``mask[token, j // 32]`` set (``mask`` ``[tokens, words]`` int32: a drafted tree, each node its
    ancestors and itself), or those up to itself without a mask: one token is a decoding step, many
    a chunk of a prompt.  A token that sees nothing gets zeros, and a row that it does not see has no effect
    on it, NaN or not.  Query head h reads kv head ``h // (heads // kv_heads)``.  ``max_new`` bounds the
    new tokens of any one sequence (``tokens`` by default); tokens past it may be left out.  Give it where it is known:
    without it a batch of many single tokens is taken for one long sequence and runs in tiles of 128 rows."""
    return _on(stream, _ops.tree_attention, q, k_cache, v_cache, table, cu, ctx, mask, max_new, scale, k_scale, v_scale, out)


def shared_attention(q, k_cache, v_cache, table, cu, ctx, groups, shared, mask=None, max_new=None, scale=None, k_scale: float = 1.0,
                     v_scale: float = 1.0, out=None, stream=None):
    """``tree_attention`` of a batch in which groups of neighbouring sequences begin with the same rows, which are read once
    for a group: a system prompt, a document, the prompt of a beam search.

    ``groups`` ``[count + 1]`` int32, not descending, delimits them: group g is the sequences ``groups[g]`` to
    ``groups[g + 1] - 1`` (sequences outside them share nothing), and their tables begin with the same pages for
    ``shared[g]`` rows at least (``shared`` ``[count]`` int32; more than one of them has cached counts as its ``ctx``).  The rows that a
    group shares are read through the table of any of its sequences.  Without matrix-core operands (``head_dim`` 64, 96, 128
    or 256, pages of 16 rows and more, 16-byte aligned tensors) every sequence reads all of its rows."""
    return _on(stream, _ops.shared_attention, q, k_cache, v_cache, table, cu, ctx, groups, shared, mask, max_new, scale, k_scale, v_scale, out)


def weighted_attention(q, k_cache, v_cache, table, cu, ctx, weights, weights_out=None, mask=None, max_new=None, scale=None,
                       k_scale: float = 1.0, v_scale: float = 1.0, out=None, stream=None):
    """``tree_attention``, and what every row was worth: ``(out, weights_out)``.

    ``weights`` ``[batch, kv_heads, rows]`` float32 holds each sequence's sums of softmax weights (any strides with the rows
    contiguous; one such tensor for a layer).  Row j of a sequence gets, for each kv head, the weights that the kv head's
    query heads give it, added up over the call's new tokens: on top of its sum where it is cached, a sum of its own where
    it is new.  ``weights_out`` (``weights`` itself by default, otherwise a tensor that does not overlap it) takes the sums of all
    rows that the sequences then have; the entries behind them are left as they are.  Rows that ``weights`` has no place for have no sum."""
    return _on(stream, _ops.weighted_attention, q, k_cache, v_cache, table, cu, ctx, weights, weights_out, mask, max_new, scale, k_scale,
               v_scale, out)


def evict(k_cache, v_cache, table, ctx, weights, fresh, keep: int, recent: int = 0, sinks: int = 0, stream=None):
    """``(table, ctx, weights)`` of the sequences after those of more than ``keep`` rows are cut to ``keep``: in every layer and
    kv head the first ``sinks`` rows, the last ``recent``, and of the others those of the largest ``weights`` ``[layers, batch,
    kv_heads, rows]`` float32 (equal ones go to the lower row; NaN counts as -inf, as does a row that ``weights`` has no place for).

    The kept rows are copied, in their order, from ``k_cache`` and ``v_cache`` ``[layers, pages, kv_heads, page_size, head_dim]``
    to the sequence's pages ``fresh`` ``[batch, ceil(keep / page_size)]`` int32, which no sequence may use; the old pages are free
    afterwards unless another sequence shares them.  A sequence of up to ``keep`` rows stays as it is, its fresh pages unused.
    Rows without a page (``-1`` in the table) are not kept: others take their places, and where there are too few of them the
    sequence gets shorter than ``keep``.
    The new table is as wide as ``table``, -1 behind a cut sequence's pages; the new weights are 0 behind its rows.  Keys keep the
    positions that they were rotated by: give ``append`` the tokens' ``positions`` from then on."""
    return _on(stream, _ops.evict, k_cache, v_cache, table, ctx, weights, fresh, keep, recent, sinks)


def commit_path(k_cache, v_cache, table, cu, ctx, path, stream=None):
    """Keeps the accepted path of each sequence's drafted tree: row ``ctx[b] + node`` of the path's j-th node becomes row
    ``ctx[b] + j`` in every layer of ``k_cache`` and ``v_cache`` ``[layers, pages, kv_heads, page_size, head_dim]``.
    ``path`` ``[batch, steps]`` int32 holds ascending nodes; entries that are none of the sequence's new tokens, as the
    -1 of padding, are passed over.  Returns the sequences' new lengths, ``ctx`` plus the path's nodes."""
    return _on(stream, _ops.commit_path, k_cache, v_cache, table, cu, ctx, path)
