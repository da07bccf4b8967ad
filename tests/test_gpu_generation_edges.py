"""GPT2Generator on the GPU: lengths at their ends, beams that end, errors of
the device."""
import numpy as np
import pytest
from test_gpu_generation import model  # noqa: F401  (the fixture: a session and its generator)

pytestmark = pytest.mark.gpu


def test_log_probs_of_the_shortest_and_the_longest_sequence(model):  # noqa: F811
    cfg, w, s, g = model
    assert g.log_probs([5]).shape == (0,)
    longest = g.log_probs(np.arange(cfg.max_pos) % cfg.vocab)
    assert longest.shape == (cfg.max_pos - 1,) and bool((longest < 0).all())


@pytest.mark.parametrize("call", ["log_probs", "generate"])
def test_an_error_of_the_device_is_raised(model, call):  # noqa: F811
    """An error that a kernel of the stream recorded (a page number out of range) ends the call, once."""
    import torch

    from tokenvector.inference_b200 import _native as N
    from tokenvector.inference_b200.generation import paged_append
    cfg, w, s, g = model
    run = {"log_probs": lambda: g.log_probs([1, 2, 3]), "generate": lambda: g.generate([[1, 2]], 2, 3)}[call]
    k = torch.zeros((2, 16, 2, 64), dtype=torch.float16, device="cuda")
    row = torch.ones((1, 2, 64), device="cuda")
    one = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    paged_append(row, row, k, k.clone(), one([[7]]), one([1]))
    with pytest.raises(N.TvqError, match="page"):
        run()
    run()


def test_weights_of_another_float_type_are_the_same_model(model):  # noqa: F811
    """The session takes embeddings and norms in any float type; so does the generator."""
    from dataclasses import replace

    import torch

    from tokenvector.inference_b200.generation import GPT2Generator
    cfg, w, s, g = model
    names = ("ln1_g", "ln1_b", "ln2_g", "ln2_b")
    wide = replace(w, wte=w.wte.astype(np.float64), wpe=w.wpe.astype(np.float64), lnf_g=w.lnf_g.astype(np.float64),
                   lnf_b=w.lnf_b.astype(np.float64),
                   layers=[{k: a.astype(np.float64) if k in names else a for k, a in L.items()} for L in w.layers])
    ids = [3, 1, 4, 1, 5, 9, 2, 6]
    assert torch.equal(GPT2Generator(s, wide).log_probs(ids), g.log_probs(ids))


def test_continuations_end_with_eos(model):  # noqa: F811
    """eos is a token of the best continuation without one: with it that continuation ends there, with its own score
    (the tolerance a token of test_gpu_generation), and the others go on."""
    from test_gpu_generation import TOL
    cfg, w, s, g = model
    prompt = np.random.default_rng(7).integers(0, cfg.vocab, 19).tolist()
    free = g.generate([prompt], 3, 20)[0]
    at = 3
    eos = free[0][0][at]
    found = g.generate([prompt], 3, 20, eos=eos)[0]
    ended = [(t, sc) for t, sc in found if t[-1] == eos and len(t) < 20]
    assert ended
    for t, sc in found:
        assert eos not in t[:-1] and (t[-1] == eos or len(t) == 20)
        own = float(g.log_probs(prompt + t)[len(prompt) - 1:].sum())
        assert abs(own - sc) <= TOL * len(t), (own, sc)
