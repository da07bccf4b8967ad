"""The paged key/value cache: writing new tokens into it and attending over it.

A layer's cache is two tensors [pages, page, kv_heads, head_dim] (float16 or
bfloat16; any strides with a contiguous last dimension, so pages may be stored
[heads, page, dim] inside and passed transposed).  Sequence s holds ctx_len[s]
tokens, token j in page table[s, j // page], slot j % page.  Its new rows are
the packed rows cu[s] .. cu[s + 1] (cu None: one row each); row i of n sits at
position ctx_len[s] - n + i.  Lengths and tables stay on the device.
"""
from __future__ import annotations

import math

import torch

from .. import _native as N
from . import _dev as D

__all__ = ["paged_append", "paged_attention"]


def _cache(k_pages, v_pages, table, ctx_len, cu, n_rows):
    """Checks the cache of one layer -> (device, type, shape array, stride array)."""
    dev = k_pages.device
    if not k_pages.is_cuda:
        raise ValueError("the cache must be on a CUDA device")
    if k_pages.dtype not in (torch.float16, torch.bfloat16) or v_pages.dtype is not k_pages.dtype:
        raise ValueError("k_pages and v_pages must both be float16 or both bfloat16")
    if k_pages.dim() != 4 or v_pages.shape != k_pages.shape:
        raise ValueError("k_pages and v_pages must be [pages, page, kv_heads, head_dim], alike")
    ks, vs = k_pages.stride(), v_pages.stride()
    if ks[3] != 1 or vs[3] != 1:
        raise ValueError("the cache's last dimension must be contiguous")
    D.check_i32(table, 2, "table")
    D.check_i32(ctx_len, 1, "ctx_len")
    seqs = ctx_len.shape[0]
    if table.shape[0] != seqs:
        raise ValueError("table must have one row for each of the %d sequences" % seqs)
    if cu is None:
        if n_rows != seqs:
            raise ValueError("without cu every sequence has one row")
    else:
        D.check_i32(cu, 1, "cu")
        if cu.shape[0] != seqs + 1:
            raise ValueError("cu must hold one entry more than there are sequences")
    D.check_dev(dev, v_pages=v_pages, table=table, ctx_len=ctx_len, cu=cu)
    return dev, D.TYPES[k_pages.dtype], D.i64s(*k_pages.shape), D.i64s(*ks[:3], *vs[:3])


def _rows(t, heads, dim, name):
    if t.dim() != 3 or (heads is not None and t.shape[1] != heads) or t.shape[2] != dim:
        raise ValueError("%s must be [rows, heads, head_dim] like the cache" % name)
    if t.stride(2) != 1:
        raise ValueError("%s must be contiguous in its last dimension" % name)


_appends, _attentions = D.Forms(), D.Forms()


def _append_form(k, v, k_pages, v_pages, table, ctx_len, cu, q):
    dev, kind, shape, strides = _cache(k_pages, v_pages, table, ctx_len, cu, k.shape[0])
    heads, dim = k_pages.shape[2:]
    _rows(k, heads, dim, "k")
    _rows(v, heads, dim, "v")
    if k.dtype not in D.TYPES or v.dtype is not k.dtype or v.shape[0] != k.shape[0]:
        raise ValueError("k and v must be float32, float16 or bfloat16 rows, alike")
    q_heads, qs = 0, (0, 0)
    if q is not None:
        _rows(q, None, dim, "q")
        if q.dtype is not k.dtype or q.shape[0] != k.shape[0]:
            raise ValueError("q must have k's type and rows")
        q_heads, qs = q.shape[1], q.stride()[:2]
    D.check_dev(dev, k=k, v=v, q=q)
    return (dev, kind, D.TYPES[k.dtype], D.i64s(*k.stride()[:2], *v.stride()[:2], *qs), q_heads, shape, strides,
            table.stride(0), table.shape[1], ctx_len.shape[0], k.shape[0])


def paged_append(k, v, k_pages, v_pages, table, ctx_len, cu=None, *, q=None):
    """Write the new rows k, v [rows, kv_heads, head_dim] (float32, float16 or
    bfloat16; strided rows of a projection's output will do) into the cache,
    rounded once to its type.  q [rows, heads, head_dim] of the same type as k
    is rounded with them and returned contiguous (None without q).  ctx_len
    counts the new tokens already."""
    key = (D.form(k), D.form(v), D.form(k_pages), D.form(v_pages), D.form(table), D.form(ctx_len), D.form(cu),
           D.form(q))
    found = _appends.get(key) or _appends.keep(key, _append_form(k, v, k_pages, v_pages, table, ctx_len, cu, q))
    dev, kind, source, src_strides, q_heads, shape, strides, table_stride, cols, seqs, n_rows = found
    q_out = None if q is None else torch.empty(q.shape, dtype=k_pages.dtype, device=dev)
    D.call("tvq_dev_paged_append", dev, kind, source, k.data_ptr(), v.data_ptr(), D.ptr(q), src_strides, q_heads,
           D.ptr(q_out), k_pages.data_ptr(), v_pages.data_ptr(), shape, strides, table.data_ptr(), table_stride, cols,
           ctx_len.data_ptr(), D.ptr(cu), seqs, n_rows, D.stream(dev))
    return q_out


def _attention_form(q, k_pages, v_pages, table, ctx_len, cu, out, max_q, window):
    n_rows = q.shape[0]
    dev, kind, shape, strides = _cache(k_pages, v_pages, table, ctx_len, cu, n_rows)
    kv_heads, dim = k_pages.shape[2:]
    _rows(q, None, dim, "q")
    heads = q.shape[1]
    if q.dtype is not k_pages.dtype:
        raise ValueError("q must have the cache's type")
    if heads % kv_heads or heads == 0:
        raise ValueError("q's heads must be a multiple of the cache's")
    if out is not None and (out.shape != q.shape or out.dtype is not q.dtype or not out.is_contiguous()):
        raise ValueError("out must be contiguous, with q's shape and type")
    if window < 0:
        raise ValueError("window must not be negative")
    D.check_dev(dev, q=q, out=out)
    most = (1 if cu is None else n_rows) if max_q is None else int(max_q)
    seqs = ctx_len.shape[0]
    with torch.cuda.device(dev):
        need = D.needed("tvq_paged_attention_workspace", heads, kv_heads, dim, seqs, n_rows, most)
    return (dev, kind, D.i64s(*q.stride()[:2]), heads, shape, strides, table.stride(0), table.shape[1], seqs, n_rows,
            most, need, 1.0 / math.sqrt(dim))


def paged_attention(q, k_pages, v_pages, table, ctx_len, cu=None, *, max_q=None, scale=None, window=0, out=None,
                    return_lse=False):
    """Causal attention of the new rows q [rows, heads, head_dim] (the cache's
    type) over the cache, which holds their own keys and values already.

    heads is a multiple of kv_heads; head h reads kv head h // (heads /
    kv_heads).  window > 0 limits a row to the last `window` keys, its own
    among them.  scale defaults to head_dim ** -0.5.  max_q: the most new rows
    of one sequence (a host number; the number of rows if not given, which is
    right but chooses the kernel for long chunks).  Returns out (written to
    `out` if given: contiguous, q's shape and type), or (out, lse) with lse
    float32 [rows, heads], the natural logarithm of the softmax's
    denominators.  A row without keys gives 0 and -inf."""
    key = (D.form(q), D.form(k_pages), D.form(v_pages), D.form(table), D.form(ctx_len), D.form(cu), D.form(out),
           max_q, window)
    found = _attentions.get(key) or _attentions.keep(key, _attention_form(q, k_pages, v_pages, table, ctx_len, cu, out,
                                                                          max_q, window))
    dev, kind, q_strides, heads, shape, strides, table_stride, cols, seqs, n_rows, most, need, root = found
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    lse = torch.empty((n_rows, heads), dtype=torch.float32, device=dev) if return_lse else None
    stream = D.stream(dev)
    ws = D.workspace("paged_attention", dev, stream, need)
    D.call("tvq_dev_paged_attention", dev, kind, q.data_ptr(), q_strides, heads, k_pages.data_ptr(),
           v_pages.data_ptr(), shape, strides, table.data_ptr(), table_stride, cols, ctx_len.data_ptr(), D.ptr(cu), seqs,
           n_rows, most, root if scale is None else scale, window, out.data_ptr(), D.ptr(lse), D.ptr(ws), need, stream)
    return (out, lse) if return_lse else out
