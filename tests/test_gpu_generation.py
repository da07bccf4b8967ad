"""Beam search with the INT8 GPT-2 stack over the paged cache.

The search is checked against a plain beam search on the host whose
log-probabilities come from the generator's own whole-sequence pass, and that
pass against the device session, whose attention is f32.  Tolerances: one
sequence's rows differ from the session's by the cache's float16 rounding
(2^-11 of K, V, q and the weights), which moves int8 activations across a
rounding boundary now and then; one such step is one 127th of an activation's
range, and the session's own tests allow 5e-2 in a logit for it, with the embedding
(the LM head) of the initial model; it is eight times as wide here.  A log-probability
has two such errors (its logit and the normaliser): 2 x 8 x 5e-2.  Between one token at
a time and the whole sequence at once only the order of f32 sums differs: rarer
steps, 0.1 a token on the whole."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

WIDE = 8
TOL_SESSION = 2 * WIDE * 5e-2
TOL = 0.1


@pytest.fixture(scope="module")
def model():
    from tokenvector.inference_b200.generation.gpt2 import GPT2Generator
    from tokenvector.inference_b200.gpt2 import GPT2Config, GPT2Session, GPT2Weights
    cfg = GPT2Config(vocab=320, d_model=128, n_heads=2, n_layers=2, d_ffn=512, max_pos=128)
    w = GPT2Weights.random(cfg, seed=5)
    for i, L in enumerate(w.layers):  # wider weights than the initial ones: the tokens depend on the context
        for k in ("attn_w", "proj_w", "fc_w", "mp_w"):
            L[k] = L[k] * 4
    w.wte = w.wte * WIDE
    s = GPT2Session(w, device=0, max_tokens=128)
    s.prepare(np.array([0, 100], np.int64))
    s.calibrate(np.random.default_rng(1).integers(0, cfg.vocab, 100))
    yield cfg, w, s, GPT2Generator(s, w)
    s.close()


@pytest.mark.parametrize("n", [2, 16, 17, 63])
def test_whole_sequence_agrees_with_the_session(model, n):
    cfg, w, s, g = model
    ids = np.random.default_rng(n).integers(0, cfg.vocab, n)
    s.prepare(np.array([0, n], np.int64))
    logits = s.forward(ids).astype(np.float64)
    lp = logits - np.log(np.exp(logits - logits.max(1, keepdims=True)).sum(1, keepdims=True)) - logits.max(1, keepdims=True)
    want = lp[np.arange(n - 1), ids[1:]]
    got = g.log_probs(ids).cpu().numpy()
    assert np.abs(got - want).max() <= TOL_SESSION, np.abs(got - want).max()


@pytest.mark.parametrize("lens,beams,new", [([1], 1, 12), ([5], 3, 20), ([16, 33, 2], 4, 18), ([40, 15], 8, 33)])
def test_scores_are_the_sequences_own(model, lens, beams, new):
    cfg, w, s, g = model
    rng = np.random.default_rng(sum(lens))
    prompts = [rng.integers(0, cfg.vocab, n).tolist() for n in lens]
    for p, found in zip(prompts, g.generate(prompts, beams, new)):
        assert len(found) == beams and len({tuple(t) for t, _ in found}) == beams
        assert all(a[1] >= b[1] for a, b in zip(found, found[1:]))
        for tokens, score in found:
            assert len(tokens) == new
            own = float(g.log_probs(p + tokens)[len(p) - 1:].sum())
            assert abs(own - score) <= TOL * new, (own, score)


@pytest.mark.parametrize("beams,new,eos", [(2, 6, None), (3, 5, None), (3, 10, 17)])
def test_search_is_a_beam_search(model, beams, new, eos):
    """No continuation that a plain beam search finds is better by more than the tolerance."""
    cfg, w, s, g = model
    prompt = np.random.default_rng(7).integers(0, cfg.vocab, 19).tolist()

    def step_log_probs(seq):
        x = g._prefill([seq], 0)[4]
        import torch
        return torch.log_softmax(g._logits(x[-1:]), 1)[0].cpu().numpy()

    live = [([], 0.0)]
    for _ in range(new):
        cands = []
        for t, sc in live:
            if eos is not None and t and t[-1] == eos:
                cands.append((t, sc))
                continue
            lp = step_log_probs(prompt + t)
            best = np.argsort(-lp, kind="stable")[:beams]
            cands += [(t + [int(v)], sc + float(lp[v])) for v in best]
        cands.sort(key=lambda c: -c[1])
        live = cands[:beams]
    found = g.generate([prompt], beams, new, eos=eos)[0]
    for (_, a), (_, b) in zip(live, found):
        assert abs(a - b) <= TOL * new, (live, found)
    if eos is not None:
        assert all(eos not in t[:-1] for t, _ in found)


def test_refusals(model):
    cfg, w, s, g = model
    with pytest.raises(ValueError):
        g.generate([[1] * 120], 2, 20)
    with pytest.raises(ValueError):
        g.generate([[1], []], 2, 4)
