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
