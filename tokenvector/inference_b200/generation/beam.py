"""Beam search on the device: the choice of the next tokens, and the move of
the beams' paged caches that follows it."""
from __future__ import annotations

from ._dev import ops

__all__ = ["beam_select", "beam_reorder"]


def beam_select(logits, scores, beams, keep, *, finished=None, eos=None):
    """One step's choice.  logits [batch * beams, vocab] (float32, float16 or
    bfloat16; one row expanded over all beams will do), scores float32 [batch *
    beams] (log-probabilities so far; -inf for a beam that does not take part)
    -> (scores float32, tokens int64, parents int32), each [batch, keep], best
    first.

    Each beam lists its `keep` largest logits (ties: the lowest token; NaN
    counts as -inf) with total = score + log softmax; the `keep` best of a
    request's lists are chosen, ties to the lower beam, then to the place in
    its list.  parents are beams of the request (0 .. beams - 1).  A finished
    beam (bool [batch * beams]) has the one continuation `eos` at no cost."""
    return ops.beam_select(logits, scores, beams, keep, finished, eos)


def beam_reorder(table, lens, parents, refs, k_pages, v_pages):
    """The beams' caches after a choice: row r of the new table continues row
    parents[r] of the old one (-1: an empty row), with room for one more token.

    table int32 [rows, cols] (or one row expanded), lens int32 [rows] (below 0
    counts as 0), parents int32 [new_rows], refs int32 [pages] (how often the tables, and whoever else keeps pages,
    hold each page), k_pages and v_pages the cache of every layer [layers,
    pages, page, kv_heads, head_dim].  Full pages are shared.  A part-filled
    last page stays with the lowest row that has it, if nobody but the old
    tables holds it, and none of their rows as a full page; the other rows take
    a free page and its filled tokens are copied (in k_pages and v_pages themselves, in every layer).  Behind a full
    page comes a free page.  Free are the pages with refs 0 before the call,
    the lowest first.  Returns (table, lens, refs, status), all new; status
    int32 [2] = (pages taken, rows left without room: their next entry is -1)."""
    return ops.beam_reorder(table, lens, parents, refs, k_pages, v_pages)
