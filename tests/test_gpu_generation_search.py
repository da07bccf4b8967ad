"""GPT2Generator.generate, token by token: a model whose logits are exact.

The stack is replaced by one that tells what the cache holds.  The value of a
token is a code of zeros and ones that depends on the token and its position;
with queries of zeros attention gives the mean of the codes of a row's whole
history, from which their sum comes back exactly (at most 96 codes: the mean's
rounding to bfloat16 is 96 2^-9 < 1/4 in the sum at most), and the logits are a
pseudo-random function of that sum, 211 of them spread over 1024 on a grid of 1/64.  A page that is shared,
copied or freed wrongly, a finished beam or a parent that is taken wrongly gives
other tokens.  The search is compared with one in 64 bits on the host: the same
tokens, and scores within the f32 error of their sums, which is 2^-22 (|score| +
|x - max| + |z|) + 2^-20 a step, of terms below 2^8 together: less than 2^-13.  At every step the worst
candidate that is taken and the best that is not are apart by more than twice
the sum of those errors, or the case would not be fit for the comparison."""
import numpy as np
import pytest

VOCAB, D, POS = 211, 128, 96
STEP_TOL = 2.0 ** -13


class Codes:
    """The model, on the host."""

    def __init__(self, seed, eos=None, pull=0.0):
        rng = np.random.default_rng(seed)
        self.code = rng.integers(0, 2, (VOCAB, POS, D)).astype(np.int64)
        self.mix = rng.integers(1, 1 << 20, (D, VOCAB)).astype(np.int64)
        self.bias = np.zeros(VOCAB)
        if eos is not None:
            self.bias[eos] = pull

    def logits(self, total):
        return (total @ self.mix % 65521) / 64.0 + self.bias

    def of(self, ids):
        return self.logits(self.code[ids, np.arange(len(ids))].sum(0))


def search(m, prompt, beams, new, eos):
    """(continuations with their scores, best first; the smallest margin; steps until all had ended; the largest terms)."""
    live, margin, ended, terms = [((), 0.0)], np.inf, None, 0.0
    for step in range(new):
        cands = []
        for t, sc in live:
            if eos is not None and eos in t:
                cands.append((t, sc))
                continue
            x = m.of(list(prompt) + list(t))
            x = x - x.max()
            z = np.log(np.exp(x).sum())
            cands += [(t + (int(v),), sc + x[v] - z) for v in np.argsort(-x, kind="stable")[:beams]]
        cands.sort(key=lambda c: -c[1])
        if len(cands) > beams:
            margin = min(margin, cands[beams - 1][1] - cands[beams][1])
        live = cands[:beams]
        terms = max(terms, -live[-1][1] + 8)  # |score| + |x - max| + |z| of what is taken, z below ln 211
        if ended is None and eos is not None and all(eos in t for t, _ in live):
            ended = step + 1
    return live, margin, ended, terms


CASES = [  # prompt lengths, beams, new tokens, page, eos, its pull, seed
    ([5], 1, 12, 8, None, 0.0, 0),
    ([1, 16, 33], 4, 40, 16, None, 0.0, 0),
    ([8, 7, 9], 8, 33, 8, None, 0.0, 26),
    ([40, 3], 5, 30, 16, 17, 300.0, 0),
    ([16, 32, 5, 24], 4, 40, 8, 0, 700.0, 5),
    ([30], 8, 20, 32, 210, 1000.0, 6),
    ([12, 1], 3, 1, 16, 9, 700.0, 1),
]


def expected(case):
    lens, beams, new, page, eos, pull, seed = case
    m = Codes(seed, eos, pull)
    rng = np.random.default_rng(seed + 100)
    prompts = [rng.integers(0, VOCAB, n).tolist() for n in lens]
    return m, prompts, [search(m, p, beams, new, eos) for p in prompts]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_cases_are_fit_for_the_comparison(case):
    lens, beams, new, page, eos, pull, seed = case
    m, prompts, want = expected(case)
    assert all(margin > 2 * new * STEP_TOL for _, margin, _, _ in want), [w[1] for w in want]
    assert all(terms < 256 for _, _, _, terms in want), [w[3] for w in want]


def test_cases_reach_what_they_stand_for():
    """Beams that had ended while others went on, and all beams of every prompt ended long before the last step."""
    some = early = 0
    for case in CASES:
        if case[4] is not None:
            want = expected(case)[2]
            some += any(len({len(t) for t, _ in found}) > 1 for found, _, _, _ in want)
            early += all(ended is not None and ended + 9 < case[2] for _, _, ended, _ in want)
    assert some and early


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_generate_finds_the_same_tokens(case, kind):
    import torch

    from tokenvector.inference_b200.generation import GPT2Generator, paged_append, paged_attention
    from tokenvector.inference_b200.gpt2 import GPT2Config
    lens, beams, new, page, eos, pull, seed = case
    m, prompts, want = expected(case)
    dev = torch.device("cuda", 0)
    code = torch.from_numpy(m.code).to(dev)
    mix, bias = torch.from_numpy(m.mix).double().to(dev), torch.from_numpy(m.bias).to(dev)

    class Told(GPT2Generator):
        def __init__(self):
            self.cfg = GPT2Config(vocab=VOCAB, d_model=D, n_heads=2, n_layers=2, d_ffn=4 * D, max_pos=POS)
            self.page, self.dtype, self.dev = page, getattr(torch, kind), dev

        def _rows(self, ids, pos, cache, table, ctx, cu, max_q):
            rows = code[ids, pos].float().view(-1, 2, D // 2)
            told = []
            for li in range(2):
                k, v = cache[0][li], cache[1][li]
                q = paged_append(torch.zeros_like(rows), rows, k, v, table, ctx, cu, q=torch.zeros_like(rows))
                mean = paged_attention(q, k, v, table, ctx, cu, max_q=max_q).view(-1, D).double()
                told.append((mean * (pos + 1)[:, None]).round())
            assert torch.equal(told[0], told[1])
            return told[1]

        def _logits(self, x):
            return ((x @ mix).remainder(65521) / 64.0 + bias).float()

    for got, (found, _, _, _) in zip(Told().generate(prompts, beams, new, eos=eos), want):
        assert [s for _, s in got] == sorted((s for _, s in got), reverse=True)
        scores = {tuple(t): s for t, s in got}
        cut = [(t[:t.index(eos) + 1] if eos is not None and eos in t else t, s) for t, s in found]
        assert set(scores) == {t for t, _ in cut}
        for t, s in cut:
            assert abs(scores[t] - s) <= new * STEP_TOL, (t, s, scores[t])
