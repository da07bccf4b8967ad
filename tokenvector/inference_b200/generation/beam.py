"""Beam search on the device: the choice of the next tokens, and the move of
the beams' paged caches that follows it."""
from __future__ import annotations

import torch

from .. import _native as N
from . import _dev as D

__all__ = ["beam_select", "beam_reorder"]


_selects, _reorders = D.Forms(), D.Forms()


def _select_form(logits, scores, beams, keep, finished, eos):
    if logits.dim() != 2 or logits.dtype not in D.TYPES or not logits.is_cuda:
        raise ValueError("logits must be a [rows, vocab] tensor of floats on a CUDA device")
    rows, vocab = logits.shape
    if beams < 1 or rows % beams:
        raise ValueError("logits must have batch * beams rows")
    if vocab > 1 and logits.stride(1) != 1:
        raise ValueError("logits must be contiguous in the vocabulary")
    if scores.dtype is not torch.float32 or scores.shape != (rows,) or not scores.is_contiguous():
        raise ValueError("scores must be float32, one for each row of logits")
    if keep > vocab:
        raise ValueError("keep larger than the vocabulary")
    if finished is not None:
        if finished.dtype is not torch.bool or finished.shape != (rows,) or not finished.is_contiguous():
            raise ValueError("finished must be bool, one for each row of logits")
        if eos is None:
            raise ValueError("finished beams need eos")
    dev = logits.device
    D.check_dev(dev, scores=scores, finished=finished)
    batch = rows // beams
    with torch.cuda.device(dev):
        need = D.needed("tvq_beam_select_workspace", batch, beams, keep, vocab)
    return dev, D.TYPES[logits.dtype], max(logits.stride(0), vocab), batch, vocab, -1 if eos is None else eos, need


def beam_select(logits, scores, beams, keep, *, finished=None, eos=None):
    """One step's choice.  logits [batch * beams, vocab] (float32, float16 or
    bfloat16), scores float32 [batch * beams] (log-probabilities so far; -inf
    for a beam that does not take part) -> (scores float32, tokens int64,
    parents int32), each [batch, keep], best first.

    Each beam lists its `keep` largest logits (ties: the lowest token; NaN
    counts as -inf) with total = score + log softmax; the `keep` best of a
    request's lists are chosen, ties to the lower beam, then to the place in
    its list.  parents are beams of the request (0 .. beams - 1).  A finished
    beam (bool [batch * beams]) has the one continuation `eos` at no cost."""
    key = (D.form(logits), D.form(scores), beams, keep, D.form(finished), eos)
    found = _selects.get(key) or _selects.keep(key, _select_form(logits, scores, beams, keep, finished, eos))
    dev, kind, stride, batch, vocab, end, need = found
    out = torch.empty((batch, keep), dtype=torch.float32, device=dev)
    tokens = torch.empty((batch, keep), dtype=torch.int64, device=dev)
    parents = torch.empty((batch, keep), dtype=torch.int32, device=dev)
    stream = D.stream(dev)
    ws = D.workspace("beam_select", dev, stream, need)
    D.call("tvq_dev_beam_select", dev, kind, logits.data_ptr(), stride, scores.data_ptr(), D.ptr(finished), batch, beams,
           keep, vocab, end, out.data_ptr(), tokens.data_ptr(), parents.data_ptr(), D.ptr(ws), need, stream)
    return out, tokens, parents


def _reorder_form(table, lens, parents, refs, k_pages, v_pages):
    D.check_i32(table, 2, "table")
    D.check_i32(lens, 1, "lens")
    D.check_i32(parents, 1, "parents")
    D.check_i32(refs, 1, "refs")
    dev = table.device
    if not table.is_cuda:
        raise ValueError("the tables must be on a CUDA device")
    if lens.shape[0] != table.shape[0]:
        raise ValueError("lens must have one entry for each row of the table")
    if k_pages.dim() != 5 or v_pages.shape != k_pages.shape or k_pages.dtype not in (torch.float16, torch.bfloat16) \
            or v_pages.dtype is not k_pages.dtype:
        raise ValueError("k_pages and v_pages must be [layers, pages, page, kv_heads, head_dim], both float16 or "
                         "both bfloat16")
    layers, pages, page, heads, dim = k_pages.shape
    ks, vs = k_pages.stride(), v_pages.stride()
    if ks[4] != 1 or vs[4] != 1:
        raise ValueError("the cache's last dimension must be contiguous")
    if refs.shape[0] != pages:
        raise ValueError("refs must have one entry for each page")
    D.check_dev(dev, lens=lens, parents=parents, refs=refs, k_pages=k_pages, v_pages=v_pages)
    rows, cols = table.shape
    new_rows = parents.shape[0]
    with torch.cuda.device(dev):
        need = D.needed("tvq_beam_reorder_workspace", pages, rows, new_rows)
    return (dev, max(table.stride(0), cols), rows, cols, new_rows, pages, D.i64s(pages, page, heads, dim, layers),
            D.i64s(*ks[:4], *vs[:4]), need)


def beam_reorder(table, lens, parents, refs, k_pages, v_pages):
    """The beams' caches after a choice: row r of the new table continues row
    parents[r] of the old one (-1: an empty row), with room for one more token.

    table int32 [rows, cols], lens int32 [rows], parents int32 [new_rows],
    refs int32 [pages] (how often the tables, and whoever else keeps pages,
    hold each page), k_pages and v_pages the cache of every layer [layers,
    pages, page, kv_heads, head_dim].  Full pages are shared.  A part-filled
    last page stays with the lowest row that has it, if nobody but the old
    tables holds it; the other rows take a free page and its filled tokens are
    copied (in k_pages and v_pages themselves, in every layer).  Behind a full
    page comes a free page.  Free are the pages with refs 0 before the call,
    the lowest first.  Returns (table, lens, refs, status), all new; status
    int32 [2] = (pages taken, rows left without room: their next entry is -1)."""
    key = (D.form(table), D.form(lens), D.form(parents), D.form(refs), D.form(k_pages), D.form(v_pages))
    found = _reorders.get(key) or _reorders.keep(key, _reorder_form(table, lens, parents, refs, k_pages, v_pages))
    dev, table_stride, rows, cols, new_rows, pages, shape, strides, need = found
    new_table = torch.empty((new_rows, cols), dtype=torch.int32, device=dev)
    new_lens = torch.empty(new_rows, dtype=torch.int32, device=dev)
    new_refs = torch.empty(pages, dtype=torch.int32, device=dev)
    status = torch.empty(2, dtype=torch.int32, device=dev)
    stream = D.stream(dev)
    ws = D.workspace("beam_reorder", dev, stream, need)
    D.call("tvq_dev_beam_reorder", dev, table.data_ptr(), table_stride, lens.data_ptr(), rows, cols, parents.data_ptr(),
           new_rows, refs.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), shape, strides, new_table.data_ptr(),
           new_lens.data_ptr(), new_refs.data_ptr(), status.data_ptr(), D.ptr(ws), need, stream)
    return new_table, new_lens, new_refs, status
