"""A paged key/value cache: appending new tokens, attention over it, and committing drafted tokens.

For batches of sequences whose rows live in pages of one pool.  The caller owns every tensor:

* a layer's cache is a K and a V tensor ``[pages, kv_heads, page_size, head_dim]`` (float16, bfloat16 or
  float8_e4m3fn; any strides with ``head_dim`` contiguous, so that K and V may share one tensor);
* ``table`` ``[batch, width]`` int32 holds each sequence's page ids, ``ctx`` ``[batch]`` int32 the rows it has;
* ``cu`` ``[batch + 1]`` int32 delimits the new tokens, which are concatenated: sequence b has tokens
  ``cu[b]`` to ``cu[b + 1] - 1``, and they take its rows ``ctx[b]``, ``ctx[b] + 1``, ...

A decoding step of a model calls, per layer, ``append`` and ``tree_attention``; a step with drafted
tokens ends with one ``commit_path`` over all layers.  Every call is asynchronous on ``stream`` (the
current one by default) and can be captured into a graph.  The indices are read on the device: a row whose
page is outside the table or the pool is not written, copied or seen.
"""

from __future__ import annotations

import struct

import torch

import qmm

_CODE = {torch.float16: qmm.DTYPE_F16, torch.bfloat16: qmm.DTYPE_BF16, torch.float8_e4m3fn: qmm.DTYPE_E4M3,
         torch.float32: qmm.DTYPE_F32}
# the C structures as packed bytes: filling a ctypes.Structure field by field costs a decode step's call several us
_KV = struct.Struct("@5P9q8i2f")
_NEW = struct.Struct("@5P8q5if")
_QUERY = struct.Struct("@3P5q5if")
_lib = qmm.lib()


def _require(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def _ints(t, name, shape, device):
    """Checks an int32 index tensor (last dimension contiguous)."""
    if t.dtype != torch.int32 or t.device != device or t.dim() != len(shape) or (t.numel() > 0 and t.stride(-1) != 1):
        raise ValueError(f"{name} must be an int32 tensor of {len(shape)} dimension(s) on the cache's device, its last one contiguous")
    for have, want in zip(t.shape, shape):
        if want is not None and have != want:
            raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple('any' if s is None else s for s in shape)}")


def _kv_bytes(k_cache, v_cache, table, cu, ctx, k_scale, v_scale, layered):
    """The packed qmm_paged_kv of checked arguments."""
    dims = 5 if layered else 4
    shape = k_cache.shape
    if len(shape) != dims or v_cache.shape != shape:
        raise ValueError("k_cache and v_cache must be alike: " + ("[layers, " if layered else "[") + "pages, kv_heads, page_size, head_dim]")
    dtype, device = k_cache.dtype, k_cache.device
    if dtype not in _CODE or dtype == torch.float32 or v_cache.dtype != dtype:
        raise ValueError("k_cache and v_cache must both be float16, bfloat16 or float8_e4m3fn")
    if device.type != "cuda" or v_cache.device != device:
        raise ValueError("k_cache and v_cache must be on one GPU")
    ks, vs = k_cache.stride(), v_cache.stride()
    if ks[-1] != 1 or vs[-1] != 1:
        raise ValueError("head_dim must be contiguous in k_cache and v_cache")
    batch = ctx.shape[0] if ctx.dim() else 0
    _ints(ctx, "ctx", (None,), device)
    _ints(table, "table", (batch, None), device)
    if cu is not None:
        _ints(cu, "cu", (batch + 1,), device)
    if not layered:
        shape, ks, vs = (1,) + tuple(shape), (0,) + ks, (0,) + vs
    layers, pages, heads, page, dim = shape
    return _KV.pack(k_cache.data_ptr(), v_cache.data_ptr(), table.data_ptr(), 0 if cu is None else cu.data_ptr(), ctx.data_ptr(),
                    table.stride(0), ks[0], ks[1], ks[2], ks[3], vs[0], vs[1], vs[2], vs[3], table.shape[1], batch, _CODE[dtype],
                    layers, pages, heads, page, dim, k_scale, v_scale)


def _rows(x, name, heads, dim, dtype, device, tokens):
    """Checks new tokens [tokens, heads, dim]; returns (token stride, head stride)."""
    shape, st = x.shape, x.stride()
    if len(shape) != 3 or shape[2] != dim or (heads is not None and shape[1] != heads) or (tokens is not None and shape[0] != tokens):
        raise ValueError(f"{name} must be [tokens, heads, head_dim] = [{tokens}, {heads}, {dim}], got {tuple(shape)}")
    if x.dtype != dtype or x.device != device:
        raise ValueError(f"{name} must be {dtype} on {device}")
    if st[2] != 1:
        raise ValueError(f"head_dim must be contiguous in {name}")
    return st


def _on(device, stream):
    """The stream's handle; the caller's current device must be the tensors'."""
    if device.index != torch.cuda.current_device():
        raise ValueError(f"the tensors are on {device}, the current device is cuda:{torch.cuda.current_device()}")
    return (torch.cuda.current_stream() if stream is None else stream).cuda_stream


def _made(stream, *tensors):
    """Tensors allocated here and used on another stream than the current one stay alive for it."""
    if stream is not None:
        for t in tensors:
            t.record_stream(stream)


def append(k, v, k_cache, v_cache, table, cu, ctx, q=None, q_out=None, positions=None, freq_base: float = 10000.0,
           rotary_dim=None, neox: bool = False, k_scale: float = 1.0, v_scale: float = 1.0, stream=None):
    """Writes new tokens' keys and values ``[tokens, kv_heads, head_dim]`` into their pages, the keys rotated on
    the way, and the rotated queries ``q`` ``[tokens, heads, head_dim]`` into ``q_out`` (a new tensor by default;
    may be ``q``).  Returns ``q_out``.

    The first ``rotary_dim`` dimensions (all by default; 0: none) turn by ``position * freq_base ** (-2 i /
    rotary_dim)``, pairs ``(2i, 2i + 1)``, or ``(i, i + rotary_dim / 2)`` with ``neox``.  A token's position is its
    row in the cache unless ``positions`` ``[tokens]`` int32 says otherwise (the depth of a drafted tree's
    node).  A float8 cache stores ``value / scale``, saturated at 448; the others need a scale of 1."""
    if not k.is_cuda:
        raise ValueError("k must be on a GPU")
    kv = _kv_bytes(k_cache, v_cache, table, cu, ctx, k_scale, v_scale, False)
    device, dtype = k_cache.device, k.dtype
    _, heads, _, dim = k_cache.shape
    if dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("k, v and q must be float16 or bfloat16")
    tokens = k.shape[0]
    ks = _rows(k, "k", heads, dim, dtype, device, tokens)
    vs = _rows(v, "v", heads, dim, dtype, device, tokens)
    if positions is not None:
        _ints(positions, "positions", (tokens,), device)
    qs = qo = (0, 0, 1)
    q_heads = 0
    if q is not None:
        qs = _rows(q, "q", None, dim, dtype, device, tokens)
        q_heads = q.shape[1]
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=dtype, device=device)
            _made(stream, q_out)
        qo = _rows(q_out, "q_out", q_heads, dim, dtype, device, tokens)
    elif q_out is not None:
        raise ValueError("q_out needs q")
    new = _NEW.pack(k.data_ptr(), v.data_ptr(), 0 if q is None else q.data_ptr(), 0 if q is None else q_out.data_ptr(),
                    0 if positions is None else positions.data_ptr(), ks[0], ks[1], vs[0], vs[1], qs[0], qs[1], qo[0], qo[1],
                    tokens, q_heads, _CODE[dtype], dim if rotary_dim is None else rotary_dim, 1 if neox else 0, freq_base)
    rc = _lib.qmm_paged_append(kv, new, _on(device, stream))
    if rc:
        qmm.check(rc)
    return q_out


def tree_attention(q, k_cache, v_cache, table, cu, ctx, mask=None, max_new=None, scale=None, k_scale: float = 1.0,
                   v_scale: float = 1.0, out=None, stream=None):
    """Attention of the new tokens' queries ``[tokens, heads, head_dim]`` (rotated, and their keys and values
    appended) over the cache.  Returns ``out``, alike.

    Token i of a sequence sees the sequence's ``ctx`` cached rows and, of its new tokens j, those with bit
    ``j % 32`` of ``mask[token, j // 32]`` set (``mask`` ``[tokens, words]`` int32: a drafted tree, each node its
    ancestors and itself), or those up to itself without a mask: one token is a decoding step, many
    a chunk of a prompt.  A token that sees nothing gets zeros, and a row that it does not see has no effect
    on it, NaN or not.  Query head h reads kv head ``h // (heads // kv_heads)``.  ``max_new`` bounds the
    new tokens of any one sequence (``tokens`` by default); knowing it, a call starts fewer workgroups."""
    if not q.is_cuda:
        raise ValueError("q must be on a GPU")
    kv = _kv_bytes(k_cache, v_cache, table, cu, ctx, k_scale, v_scale, False)
    device, dtype = k_cache.device, q.dtype
    if dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("q must be float16 or bfloat16")
    dim = k_cache.shape[3]
    qs = _rows(q, "q", None, dim, dtype, device, None)
    tokens, heads = q.shape[0], q.shape[1]
    if out is None:
        out = torch.empty(q.shape, dtype=dtype, device=device)
        _made(stream, out)
    os_ = _rows(out, "out", heads, dim, dtype, device, tokens)
    words = 0
    if mask is not None:
        _ints(mask, "mask", (tokens, None), device)
        words = mask.shape[1]
    if scale is None:
        scale = 0.0
    elif scale == 0.0:
        raise ValueError("scale must not be 0")
    query = _QUERY.pack(q.data_ptr(), out.data_ptr(), mask.data_ptr() if words else 0, qs[0], qs[1], os_[0], os_[1],
                        mask.stride(0) if words else 0, tokens, tokens if max_new is None else max_new, heads, _CODE[dtype], words, scale)
    handle = _on(device, stream)
    need = _lib.qmm_paged_attention_workspace(kv, query)
    space = None
    if need:
        space = torch.empty(need, dtype=torch.uint8, device=device)  # the allocator's: safe to capture
        _made(stream, space)
    if mask is not None and not words and tokens:
        raise ValueError("mask has no words")
    rc = _lib.qmm_paged_tree_attention(kv, query, space.data_ptr() if need else None, need, handle)
    if rc:
        qmm.check(rc)
    return out


def commit_path(k_cache, v_cache, table, cu, ctx, path, stream=None):
    """Keeps the accepted path of each sequence's drafted tree: row ``ctx[b] + path[b, j]`` becomes row
    ``ctx[b] + j`` in every layer of ``k_cache`` and ``v_cache`` ``[layers, pages, kv_heads, page_size, head_dim]``.
    ``path`` ``[batch, steps]`` int32 holds ascending nodes, padded with -1.  Returns the sequences' new lengths,
    ``ctx`` plus the path's nodes."""
    if not path.is_cuda:
        raise ValueError("path must be on a GPU")
    kv = _kv_bytes(k_cache, v_cache, table, cu, ctx, 1.0, 1.0, True)
    device = k_cache.device
    batch = ctx.shape[0]
    _ints(path, "path", (batch, None), device)
    lens = torch.empty(batch, dtype=torch.int32, device=device)
    _made(stream, lens)
    rc = _lib.qmm_paged_commit_path(kv, path.data_ptr(), path.stride(0), path.shape[1], lens.data_ptr(), _on(device, stream))
    if rc:
        qmm.check(rc)
    return lens
