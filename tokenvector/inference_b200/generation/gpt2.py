"""Beam search with the INT8 GPT-2 stack: prompts through the layers once, then
a token of every beam a step, out of a paged key/value cache.

The blocks are those of the device session (LayerNorm -> int8, INT8 linears
with static activation scales, erf GELU, f32 residual stream, tied f32 LM
head), called layer by layer on device buffers, with the attention replaced by
`paged_append` and `paged_attention` over a float16 cache; `beam_select` picks
each step's tokens and `beam_reorder` moves the beams' caches after them.
Nothing of a step goes through the host, except that with `eos` every eighth
step asks whether all beams have ended.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from .. import _native as N
from . import _dev as D
from .beam import beam_reorder, beam_select
from .paged import paged_append, paged_attention

__all__ = ["GPT2Generator"]


class GPT2Generator:
    """Decoding with the INT8 linears and calibrated activation scales of a
    `GPT2Session` (its `calibrate` has run, or it was loaded from a PTQ
    artefact).  `weights`: the session's `GPT2Weights` (embeddings and
    LayerNorms are not quantized)."""

    def __init__(self, session, weights, *, page: int = 16, dtype=torch.float16):
        cfg = session.cfg
        d = cfg.d_model

        def same(a, *shape):
            if np.shape(a) != shape:
                raise ValueError("weights of another shape than the session's")
            return np.asarray(a, np.float32)

        if len(weights.layers) != cfg.n_layers:
            raise ValueError("weights of another shape than the session's")
        norms = [[same(w[name], d) for name in ("ln1_g", "ln1_b", "ln2_g", "ln2_b")] for w in weights.layers]
        final = same(weights.lnf_g, d), same(weights.lnf_b, d)
        wte, wpe = same(weights.wte, cfg.vocab, d), same(weights.wpe, cfg.max_pos, d)
        self.cfg, self.page, self.dtype = cfg, page, dtype
        self.dev = torch.device("cuda", session.device)
        put = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(self.dev)  # noqa: E731
        self.scales = put(session.act_scales())  # [layers, 4]: ln_1, attention, ln_2, GELU outputs
        self.layers = []
        for li, norm in enumerate(norms):
            lin = [tuple(put(x) for x in session.linear_i8(li, which)) + (put(session._bias[li][which]),)
                   for which in range(4)]
            self.layers.append((lin, *(put(a) for a in norm)))
        self.lnf = put(final[0]), put(final[1])
        self.wte, self.wpe = put(wte), put(wpe)
        self.head = self._split(self.wte)

    # ---- the stack on T rows
    def _call(self, name, *args):
        D.call(name, self.dev, *args, D.stream(self.dev))

    def _check(self):
        """Waits for the stream; raises what its kernels recorded (a wait that ran out, a page out of range)."""
        self._call("tvq_device_error")

    def _split(self, x):
        hi, lo = (torch.empty(x.shape, dtype=torch.float16, device=self.dev) for _ in range(2))
        scale = torch.empty(x.shape[0], dtype=torch.float32, device=self.dev)
        self._call("tvq_dev_split_f16_rows", x.data_ptr(), hi.data_ptr(), lo.data_ptr(), scale.data_ptr(), *x.shape)
        return hi, lo, scale

    def _norm(self, x, gamma, beta, scale=None):
        """LayerNorm of f32 rows: float32, or int8 under the static scale."""
        y = torch.empty(x.shape, dtype=torch.float32 if scale is None else torch.int8, device=self.dev)
        self._call("tvq_dev_layernorm", x.data_ptr(), gamma.data_ptr(), beta.data_ptr(),
                   y.data_ptr() if scale is None else None, None if scale is None else y.data_ptr(), D.ptr(scale), None,
                   *x.shape, C.c_double(self.cfg.eps))
        return y

    def _linear(self, x, lin, scale, *, residual=None, act=N.ACT_NONE, out_scale=None):
        """An INT8 linear: float32 out (+ residual), or int8 under out_scale."""
        w, sw, bias = lin
        (m, k), n = x.shape, w.shape[0]
        y = torch.empty((m, n), dtype=torch.float32 if out_scale is None else torch.int8, device=self.dev)
        self._call("tvq_dev_gemm", N.GEMM_I8, x.data_ptr(), w.data_ptr(), bias.data_ptr(), D.ptr(residual),
                   y.data_ptr() if out_scale is None else None, None if out_scale is None else y.data_ptr(), m, n, k,
                   scale.data_ptr(), sw.data_ptr(), 1, act, D.ptr(out_scale), None)
        return y

    def _rows(self, ids, pos, cache, table, ctx, cu, max_q):
        """Hidden states of the new rows (token ids and positions [T]); their
        keys and values go into the cache."""
        cfg = self.cfg
        heads, dim = cfg.n_heads, cfg.d_model // cfg.n_heads
        x = self.wte[ids] + self.wpe[pos]
        for li, (lin, g1, b1, g2, b2) in enumerate(self.layers):
            s = self.scales[li]
            qkv = self._linear(self._norm(x, g1, b1, s[0:1]), lin[0], s[0:1])
            q, k, v = (t.unflatten(1, (heads, dim)) for t in qkv.split(cfg.d_model, 1))
            k_pages, v_pages = cache[0][li], cache[1][li]
            q = paged_append(k, v, k_pages, v_pages, table, ctx, cu, q=q)
            a = paged_attention(q, k_pages, v_pages, table, ctx, cu, max_q=max_q).view(-1, cfg.d_model).float()
            aq = torch.empty(a.shape, dtype=torch.int8, device=self.dev)
            self._call("tvq_dev_quantize_int8", a.data_ptr(), aq.data_ptr(), a.numel(), s[1:2].data_ptr())
            x = self._linear(aq, lin[1], s[1:2], residual=x)
            h = self._linear(self._norm(x, g2, b2, s[2:3]), lin[2], s[2:3], act=N.ACT_GELU_ERF, out_scale=s[3:4])
            x = self._linear(h, lin[3], s[3:4], residual=x)
        return x

    def _logits(self, x):
        a, w = self._split(self._norm(x, *self.lnf)), self.head
        y = torch.empty((x.shape[0], self.cfg.vocab), dtype=torch.float32, device=self.dev)
        self._call("tvq_dev_gemm_f16x3", *(t.data_ptr() for t in a + w), y.data_ptr(), x.shape[0], self.cfg.vocab,
                   self.cfg.d_model)
        return y

    # ---- prompts
    def _ids(self, prompt):
        """A prompt's token ids as int64, checked on the host: the embeddings are indexed on the device."""
        ids = np.asarray(prompt)
        if ids.ndim != 1 or ids.size == 0:
            raise ValueError("every prompt needs a token")
        if ids.dtype.kind not in "iu" or ids.min() < 0 or ids.max() >= self.cfg.vocab:
            raise ValueError("token ids must be integers within the vocabulary")
        if ids.size > self.cfg.max_pos:
            raise ValueError("sequence longer than the model's positions")
        return ids.astype(np.int64)

    def _prefill(self, prompts, spare_pages, cols=0):
        """The prompts' cache and last hidden states, with `spare_pages` free
        pages and `cols` table columns at least."""
        page, cfg = self.page, self.cfg
        prompts = [self._ids(p) for p in prompts]
        lens = [len(p) for p in prompts]
        held = [-(-n // page) for n in lens]
        pool = sum(held) + spare_pages
        shape = (cfg.n_layers, pool, page, cfg.n_heads, cfg.d_model // cfg.n_heads)
        cache = tuple(torch.empty(shape, dtype=self.dtype, device=self.dev) for _ in range(2))
        table = np.full((len(prompts), max(cols, max(held))), -1, np.int32)
        first = 0
        for s, n in enumerate(held):
            table[s, :n] = np.arange(first, first + n)
            first += n
        put = lambda a, t: torch.from_numpy(np.ascontiguousarray(a)).to(self.dev, t)  # noqa: E731
        table = put(table, torch.int32)
        refs = put((np.arange(pool) < first).astype(np.int32), torch.int32)
        cu = np.concatenate([[0], np.cumsum(lens)])
        ids = put(np.concatenate(prompts), torch.int64)
        pos = put(np.concatenate([np.arange(n) for n in lens]), torch.int64)
        ctx = put(lens, torch.int32)
        x = self._rows(ids, pos, cache, table, ctx, put(cu, torch.int32), max(lens))
        return cache, table, refs, ctx, x, put(cu, torch.int64)

    def log_probs(self, ids):
        """log p(ids[t] | ids[:t]) for t >= 1, one sequence at once: float32 [len - 1]."""
        ids = self._ids(ids)
        if ids.size == 1:  # its logits predict nothing
            return torch.empty(0, dtype=torch.float32, device=self.dev)
        x = self._prefill([ids], 0)[4]
        lp = torch.log_softmax(self._logits(x[:-1]), 1)
        lp = lp.gather(1, torch.as_tensor(ids[1:], device=self.dev)[:, None])[:, 0]
        self._check()
        return lp

    def generate(self, prompts, beams: int, max_new: int, eos: int | None = None):
        """Beam search over several prompts (lists of token ids) at once.

        Returns for each prompt its `beams` best continuations, best first, as
        (tokens, score) with score the sum of the tokens' log-probabilities;
        a continuation ends with `eos` or after max_new tokens."""
        cfg, page = self.cfg, self.page
        if max_new < 1:
            raise ValueError("max_new must be at least 1")
        longest = max(len(p) for p in prompts)
        if longest + max_new > cfg.max_pos:
            raise ValueError("prompt and continuation exceed the model's positions")
        rows = len(prompts) * beams
        cols = -(-(longest + max_new) // page) + 1
        # what the beams can hold apart from the prompts' full pages, and a page each while a step frees another
        cache, table, refs, ctx, x, cu = self._prefill(prompts, rows * (-(-max_new // page) + 3), cols)
        end = -1 if eos is None else eos
        scores, tokens, _ = beam_select(self._logits(x[cu[1:] - 1]), torch.zeros(len(prompts), device=self.dev), 1,
                                        beams, eos=None)
        # every prompt's cache becomes that of its beams
        parents = torch.arange(len(prompts), dtype=torch.int32, device=self.dev).repeat_interleave(beams)
        first_row = torch.arange(0, rows, beams, dtype=torch.int32, device=self.dev)[:, None]
        tokens, scores = tokens.view(rows), scores.view(rows)
        finished = tokens == end
        history = tokens[:, None]
        short = torch.zeros((), dtype=torch.int32, device=self.dev)
        for step in range(1, max_new):
            table, lens, refs, status = beam_reorder(table, ctx, parents, refs, *cache)
            short = torch.maximum(short, status[1])
            ctx = lens + 1  # the new token of every beam
            x = self._rows(tokens, lens.long(), cache, table, ctx, None, 1)
            new_scores, new_tokens, beam = beam_select(self._logits(x), scores, beams, beams,
                                                       finished=finished if eos is not None else None, eos=eos)
            parents = (beam + first_row).view(rows)
            tokens, scores = new_tokens.view(rows), new_scores.view(rows)
            history = torch.cat([history[parents.long()], tokens[:, None]], 1)
            finished = finished[parents.long()] | (tokens == end)
            if eos is not None and step % 8 == 0 and bool(finished.all()):
                break
        if int(short) > 0:
            raise RuntimeError("the page pool ran out")
        self._check()
        out = []
        for s in range(len(prompts)):
            mine = []
            for r in range(s * beams, (s + 1) * beams):
                t = history[r].tolist()
                mine.append((t[:t.index(end) + 1] if end in t else t, float(scores[r])))
            out.append(mine)
        return out
