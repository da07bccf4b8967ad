"""The paged key/value cache: writing new tokens into it and attending over it.

A layer's cache is two tensors [pages, page, kv_heads, head_dim] (float16 or
bfloat16; any strides with a contiguous last dimension, so pages may be stored
[heads, page, dim] inside and passed transposed).  Sequence s holds ctx_len[s]
tokens, token j in page table[s, j // page], slot j % page.  Its new rows are
the packed rows cu[s] .. cu[s + 1] (cu None: one row each); row i of n sits at
position ctx_len[s] - n + i.  Lengths and tables stay on the device.
"""
from __future__ import annotations

from ._dev import ops

__all__ = ["paged_append", "paged_attention"]


def paged_append(k, v, k_pages, v_pages, table, ctx_len, cu=None, *, q=None):
    """Write the new rows k, v [rows, kv_heads, head_dim] (float32, float16 or
    bfloat16; strided rows of a projection's output will do) into the cache,
    rounded once to its type.  q [rows, heads, head_dim] of the same type as k
    is rounded with them and returned contiguous (None without q).  ctx_len
    counts the new tokens already."""
    return ops.paged_append(k, v, k_pages, v_pages, table, ctx_len, cu, q)


def paged_attention(q, k_pages, v_pages, table, ctx_len, cu=None, *, max_q=None, scale=None, window=0, out=None,
                    return_lse=False):
    """Causal attention of the new rows q [rows, heads, head_dim] (the cache's
    type) over the cache, which holds their own keys and values already.

    heads is a multiple of kv_heads; head h reads kv head h // (heads /
    kv_heads).  window > 0 limits a row to the last `window` keys, its own
    among them.  scale defaults to head_dim ** -0.5.  max_q: the most new rows
    of one sequence (a host number; the number of rows if not given, which is
    right but chooses the kernel for long chunks; rows of a sequence behind its
    first max_q are left out).  Returns out (written to
    `out` if given: contiguous, q's shape and type), or (out, lse) with lse
    float32 [rows, heads], the natural logarithm of the softmax's
    denominators.  A row without keys gives 0 and -inf."""
    out, lse = ops.paged_attention(q, k_pages, v_pages, table, ctx_len, cu, max_q, scale, window, out, return_lse)
    return (out, lse) if return_lse else out
